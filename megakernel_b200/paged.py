"""Serving operators around a paged 8-bit key/value cache.

The parts of a serving step with drafted tokens, as hand-written sm_100a
kernels behind the C ABI (``megakernel_qk_norm_rope``, ``megakernel_kv8_*``,
``megakernel_verify_drafts`` in include/megakernel.h, which states each
operator's formula):

- ``qk_norm_rope``: RMS norm of every query and key head and their rotation;
- ``kv8_append`` / ``kv8_read``: keys and values into a paged cache of 8-bit
  codes with one scale per (page, K or V, head), and back;
- ``kv8_attend``: attention over that cache, from one row per sequence to
  whole prompts;
- ``verify_drafts``: which drafted tokens stand, and the token after them;
- ``PagedCache8``: the pools of a model's layers and the page tables.

Rows of several sequences are packed: sequence ``b`` owns rows
``starts[b]:starts[b + 1]``, the first of them at position ``first[b]``.  Rows
at negative positions are padding.  ``page_table``, ``starts`` and ``first`` are
int32 CUDA tensors; they are read by the kernels only, so a call never waits
for the GPU.  What the host can check raises ValueError at once; page ids and
positions that are out of range are left out by the kernels and reported by
``check()``.  All calls run on torch's current stream, or on ``stream``, and
may be captured into a CUDA graph (after one call outside of it).  There is no
CPU path.
"""
from __future__ import annotations

import math
import struct

import torch

from . import _lib

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
FORMATS = {torch.float8_e4m3fn: 0, torch.int8: 1}
KV_DTYPES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
PAGE_SIZES = (16, 32, 64)
HEAD_DIMS = (64, 128)

_status = {}
_work_floats = {}   # scratch of kv8_attend by what it depends on
_lib_fns = None
_get_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream
# struct mk_kv8 and mk_qk_norm_rope in C order (include/megakernel.h)
_pack_kv8 = struct.Struct("@5P3q8i").pack
_pack_norm_rope = struct.Struct("@9P8q6if4x").pack


def _fns():
    """The C entries, bound once, after the status word of the current device."""
    global _lib_fns
    if _lib_fns is None:
        L = _lib.load()
        _lib_fns = (L.megakernel_qk_norm_rope, L.megakernel_kv8_append, L.megakernel_kv8_read,
                    L.megakernel_kv8_attend, L.megakernel_verify_drafts, L.megakernel_kv8_attend_workspace)
    return _lib_fns


def _status_of(idx: int) -> int:
    """Address of device idx's status word; made (and waited for) at its first use."""
    got = _status.get(idx)
    if got is None:
        t = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
        torch.cuda.current_stream(idx).synchronize()
        got = _status[idx] = (t, t.data_ptr())
    return got[1]


def check(device=None) -> None:
    """Wait for the device and raise if a kernel of this module met metadata
    out of range since the last check (page ids, positions, row starts)."""
    dev = torch.device("cuda" if device is None else device)
    idx = torch.cuda.current_device() if dev.index is None else dev.index
    _status_of(idx)
    torch.cuda.synchronize(idx)
    t = _status[idx][0]
    rc = int(t.item())
    if rc:
        t.zero_()
        torch.cuda.synchronize(idx)
        _lib.check(rc, "paged operators")


def _elsewhere(fn, idx, stream, args, kw):
    """fn(*args, **kw) on device idx, and on `stream` if one is given; tensors
    used on a stream that is not theirs are kept until it has passed."""
    with torch.cuda.device(idx):
        if stream is None:
            return fn(*args, **kw)
        for t in (*args, *kw.values()):
            if isinstance(t, torch.Tensor) and t.is_cuda:
                t.record_stream(stream)
        with torch.cuda.stream(stream):
            return fn(*args, **kw)


def _rows(t, name):
    """Strides of a [rows, heads, head_dim] operand that is read in 16-byte
    vectors (0 for an axis of one element)."""
    if t.dim() != 3 or not t.is_cuda:
        raise ValueError(f"{name}: a CUDA tensor [rows, heads, head_dim]")
    if t.dtype not in TYPES:
        raise ValueError(f"{name}: float32, bfloat16 or float16")
    s0, s1, s2 = t.stride()
    per = 3 if t.dtype is torch.float32 else 7
    if s2 != 1 or (s0 | s1) & per or s0 < 0 or s1 < 0 or t.data_ptr() & 15:
        n, h, d = t.shape
        s0, s1 = s0 if n > 1 else 0, s1 if h > 1 else 0
        if (s2 != 1 and d > 1) or (s0 | s1) & per or s0 < 0 or s1 < 0 or t.data_ptr() & 15:
            raise ValueError(f"{name}: head_dim contiguous, rows and heads at multiples of 16 bytes")
    return s0, s1


def _vector(t, name, dtype, n, idx):
    if t.dtype is not dtype or t.get_device() != idx or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {str(dtype)[6:]} [{n}] on cuda:{idx}")


def _cache(codes, scales, page_table, starts, first, rows):
    """The checked cache arguments: (struct mk_kv8, device index, seqs, kv_heads, head_dim)."""
    if codes.dim() != 5 or not codes.is_cuda or codes.dtype not in FORMATS:
        raise ValueError("codes: CUDA float8_e4m3fn or int8 [pages, 2, kv_heads, page_size, head_dim]")
    idx = codes.get_device()
    pages, two, hk, page, d = codes.shape
    if two != 2 or page not in PAGE_SIZES or d not in HEAD_DIMS or hk < 1:
        raise ValueError(f"codes: [pages, 2, kv_heads, page_size, head_dim], page_size of {PAGE_SIZES}, head_dim of {HEAD_DIMS}")
    s0, s1, s2, s3, s4 = codes.stride()
    held = page * d
    if s4 != 1 or s3 != d or (s2 != held and hk > 1) or s1 != hk * held:
        raise ValueError("codes: a page's codes contiguous")
    page_stride = s0 if pages > 1 else 2 * hk * held
    if page_stride < 2 * hk * held or page_stride & 15 or codes.data_ptr() & 15:
        raise ValueError("codes: pages at multiples of 16 bytes, not overlapping")
    if scales.dtype is not torch.float32 or scales.get_device() != idx or tuple(scales.shape) != (pages, 2, hk):
        raise ValueError("scales: float32 [pages, 2, kv_heads] on the cache's device")
    z0, z1, z2 = scales.stride()
    scale_stride = z0 if pages > 1 else 2 * hk
    if (z2 != 1 and hk > 1) or z1 != hk or scale_stride < 2 * hk:
        raise ValueError("scales: a page's scales contiguous, pages not overlapping")
    if page_table.dim() != 2 or page_table.dtype is not torch.int32 or page_table.get_device() != idx:
        raise ValueError("page_table: int32 [seqs, pages] on the cache's device")
    b, width = page_table.shape
    t0, t1 = page_table.stride()
    table_stride = t0 if b > 1 else width
    if (t1 != 1 and width > 1) or table_stride < width:
        raise ValueError("page_table: a sequence's pages contiguous, rows not overlapping")
    _vector(starts, "starts", torch.int32, b + 1, idx)
    _vector(first, "first", torch.int32, b, idx)
    return (_pack_kv8(codes.data_ptr(), scales.data_ptr(), page_table.data_ptr(), starts.data_ptr(), first.data_ptr(),
                      page_stride, scale_stride, table_stride, pages, width, hk, page, d, FORMATS[codes.dtype], b, rows),
            idx, b, hk, d)


def qk_norm_rope(q, k, q_gain, k_gain, cos, sin, positions, *, eps=1e-6, q_out=None, k_out=None, stream=None):
    """RMS norm and rotation of every head of q [rows, q_heads, D] and k
    [rows, kv_heads, D] in one pass; returns (q_out, k_out).

    q, k, the gains [D] and the outputs share a dtype; q and k may be slices
    of one packed projection, and an output may be its input.  cos, sin: fp32
    tables [positions, D / 2]; positions: int32 [rows].  D 64 or 128.  A row
    whose position is outside the tables is not written (see ``check``)."""
    q_row, q_head = _rows(q, "q")
    k_row, k_head = _rows(k, "k")
    idx = q.get_device()
    if stream is not None or idx != _get_device():
        return _elsewhere(qk_norm_rope, idx, stream, (q, k, q_gain, k_gain, cos, sin, positions),
                          dict(eps=eps, q_out=q_out, k_out=k_out))
    dtype = q.dtype
    rows, hq, d = q.shape
    k_rows, hk, k_d = k.shape
    if k_rows != rows or k_d != d or k.dtype is not dtype or k.get_device() != idx:
        raise ValueError("k: q's rows, head_dim, dtype and device")
    if d not in HEAD_DIMS:
        raise ValueError(f"head_dim: one of {HEAD_DIMS}")
    _vector(q_gain, "q_gain", dtype, d, idx)
    _vector(k_gain, "k_gain", dtype, d, idx)
    size, half = cos.shape if cos.dim() == 2 else (0, 0)
    if half != d // 2 or cos.shape != sin.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32 \
            or cos.get_device() != idx or sin.get_device() != idx or not cos.is_contiguous() or not sin.is_contiguous():
        raise ValueError(f"cos, sin: contiguous float32 [positions, {d // 2}] on q's device")
    if (q_gain.data_ptr() | k_gain.data_ptr() | cos.data_ptr() | sin.data_ptr()) & 15:
        raise ValueError("q_gain, k_gain, cos, sin: 16-byte aligned")
    _vector(positions, "positions", torch.int32, rows, idx)
    if not eps >= 0.0:
        raise ValueError("eps: not negative")
    if q_out is None:
        q_out = q.new_empty((rows, hq, d))
        qo_row, qo_head = hq * d, d
    else:
        qo_row, qo_head = _rows(q_out, "q_out")
        if q_out.shape != q.shape or q_out.dtype is not dtype or q_out.get_device() != idx:
            raise ValueError("q_out: the shape, dtype and device of q")
    if k_out is None:
        k_out = k.new_empty((rows, hk, d))
        ko_row, ko_head = hk * d, d
    else:
        ko_row, ko_head = _rows(k_out, "k_out")
        if k_out.shape != k.shape or k_out.dtype is not dtype or k_out.get_device() != idx:
            raise ValueError("k_out: the shape, dtype and device of k")
    rc = _fns()[0](_pack_norm_rope(q.data_ptr(), k.data_ptr(), q_gain.data_ptr(), k_gain.data_ptr(), q_out.data_ptr(),
                                   k_out.data_ptr(), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), q_row, q_head,
                                   k_row, k_head, qo_row, qo_head, ko_row, ko_head, size, rows, hq, hk, d, TYPES[dtype],
                                   eps), _status_of(idx), _raw_stream(idx))
    if rc:
        _lib.check(rc, "megakernel_qk_norm_rope")
    return q_out, k_out


def kv8_append(codes, scales, k, v, page_table, starts, first, *, stream=None):
    """Quantise k and v [rows, kv_heads, D] into the cache at their rows' positions.

    A page's scale is the smallest power of two that fits the magnitudes
    written to it; a page that already holds earlier positions keeps the larger
    of its scale and the new one, its earlier codes rounded again if that grows.
    ``codes`` and ``scales`` are updated in place.  No two sequences of a call
    may write to one page."""
    k_row, k_head = _rows(k, "k")
    v_row, v_head = _rows(v, "v")
    rows, heads, dim = k.shape
    cache, idx, _, hk, d = _cache(codes, scales, page_table, starts, first, rows)
    if k.shape != v.shape or heads != hk or dim != d or k.dtype is not v.dtype or k.get_device() != idx \
            or v.get_device() != idx:
        raise ValueError("k, v: one shape [rows, kv_heads, head_dim] and dtype, on the cache's device")
    if stream is not None or idx != _get_device():
        return _elsewhere(kv8_append, idx, stream, (codes, scales, k, v, page_table, starts, first), {})
    rc = _fns()[1](cache, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head, TYPES[k.dtype], _status_of(idx),
                   _raw_stream(idx))
    if rc:
        _lib.check(rc, "megakernel_kv8_append")


def kv8_read(codes, scales, page_table, starts, first, rows, *, dtype=torch.bfloat16, stream=None):
    """The cached keys and values of the rows' positions: (k, v), each
    [rows, kv_heads, D] of `dtype`.  rows: starts[-1], as a number."""
    if rows < 0:
        raise ValueError("rows: not negative")
    if dtype not in TYPES:
        raise ValueError("dtype: float32, bfloat16 or float16")
    cache, idx, _, hk, d = _cache(codes, scales, page_table, starts, first, rows)
    if stream is not None or idx != _get_device():
        return _elsewhere(kv8_read, idx, stream, (codes, scales, page_table, starts, first, rows), dict(dtype=dtype))
    k, v = scales.new_empty((2, rows, hk, d), dtype=dtype).unbind(0)
    rc = _fns()[2](cache, k.data_ptr(), v.data_ptr(), TYPES[dtype], _status_of(idx), _raw_stream(idx))
    if rc:
        _lib.check(rc, "megakernel_kv8_read")
    return k, v


def kv8_attend(q, codes, scales, page_table, starts, first, *, kv_lens=None, sm_scale=None, causal=True, window=0,
               out=None, return_lse=False, stream=None):
    """Attention of q [rows, q_heads, D] (bf16 or f16) over the cache.

    A row at position p of sequence b sees the positions j < kv_lens[b]
    (default: up to the sequence's last row), with ``causal`` also j <= p, with
    ``window`` > 0 also j > p - window.  Query head h reads key/value head
    h // (q_heads // kv_heads).  sm_scale defaults to D ** -0.5.  Returns out
    [rows, q_heads, D] of q's dtype, and with ``return_lse`` the fp32
    log-sum-exp [rows, q_heads]; a row that sees nothing gives 0 and -inf."""
    q_row, q_head = _rows(q, "q")
    rows, hq, q_d = q.shape
    cache, idx, seqs, hk, d = _cache(codes, scales, page_table, starts, first, rows)
    if q.dtype is torch.float32 or q.get_device() != idx or q_d != d:
        raise ValueError("q: bfloat16 or float16 [rows, q_heads, head_dim] on the cache's device")
    if hq < 1 or hq % hk:
        raise ValueError("q_heads: a multiple of kv_heads")
    if seqs == 0 and rows > 0:
        raise ValueError("rows without a sequence")
    if kv_lens is not None:
        _vector(kv_lens, "kv_lens", torch.int32, seqs, idx)
    if window < 0:
        raise ValueError("window: not negative")
    if sm_scale is None:
        sm_scale = d ** -0.5
    elif not 0.0 < sm_scale < math.inf:
        raise ValueError("sm_scale: positive")
    if out is not None and (out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != idx
                            or not out.is_contiguous() or out.data_ptr() & 15):
        raise ValueError("out: contiguous, of q's shape, dtype and device")
    if stream is not None or idx != _get_device():
        return _elsewhere(kv8_attend, idx, stream, (q, codes, scales, page_table, starts, first),
                          dict(kv_lens=kv_lens, sm_scale=sm_scale, causal=causal, window=window, out=out,
                               return_lse=return_lse))
    if out is None:
        out = q.new_empty((rows, hq, d))
    lse = scales.new_empty((rows, hq)) if return_lse else None
    key = (idx, codes.dtype, codes.shape[3], d, hk, hq)
    floats = _work_floats.get(key)
    if floats is None:
        floats = _fns()[5](cache, hq)
        if floats < 0:
            _lib.check(floats, "megakernel_kv8_attend_workspace")
        if rows and seqs:
            _work_floats[key] = floats = -(-floats // 4)
    work = scales.new_empty((floats,))
    rc = _fns()[3](cache, q.data_ptr(), q_row, q_head, hq, TYPES[q.dtype], sm_scale, 1 if causal else 0, window,
                   None if kv_lens is None else kv_lens.data_ptr(), out.data_ptr(),
                   None if lse is None else lse.data_ptr(), work.data_ptr(), 4 * floats, _status_of(idx),
                   _raw_stream(idx))
    if rc:
        _lib.check(rc, "megakernel_kv8_attend")
    return (out, lse) if return_lse else out


def verify_drafts(tokens, target_probs, draft_probs, uniforms, sample_u, starts, *, stream=None):
    """Which drafted tokens stand, and the token after them: (out, accepted).

    Row i of sequence b was fed tokens[starts[b] + i] (row 0: the last confirmed
    token, then the drafts).  target_probs fp32 [rows, vocab]: the target's
    probabilities after each row; draft_probs (same shape, or None for drafts
    that were certain): what the next row's draft was picked from.  uniforms
    [rows] (entry i decides on draft i + 1) and sample_u [seqs] are random
    numbers in [0, 1).  out int32 [rows]: per sequence the kept drafts, the
    drawn token, then -1; accepted int32 [seqs].  The arithmetic is in whole
    numbers (units of 2^-36 and 2^-24), so results are exact and repeatable."""
    if target_probs.dim() != 2 or not target_probs.is_cuda or target_probs.dtype is not torch.float32:
        raise ValueError("target_probs: CUDA float32 [rows, vocab]")
    rows, vocab = target_probs.shape
    idx = target_probs.get_device()
    if vocab < 1 or starts.dim() != 1 or starts.numel() < 1:
        raise ValueError("vocab: at least one token; starts: int32 [seqs + 1]")
    seqs = starts.numel() - 1
    _vector(starts, "starts", torch.int32, seqs + 1, idx)
    _vector(tokens, "tokens", torch.int32, rows, idx)
    _vector(uniforms, "uniforms", torch.float32, rows, idx)
    _vector(sample_u, "sample_u", torch.float32, seqs, idx)
    t0, t1 = target_probs.stride()
    d0, d1 = vocab, 1
    if draft_probs is not None:
        if draft_probs.shape != target_probs.shape or draft_probs.dtype is not torch.float32 \
                or draft_probs.get_device() != idx:
            raise ValueError("draft_probs: float32, of target_probs' shape and device")
        d0, d1 = draft_probs.stride()
    if rows <= 1:
        t0 = d0 = vocab
    if ((t1 != 1 or d1 != 1) and vocab > 1) or t0 < vocab or d0 < vocab:
        raise ValueError("probabilities: vocab contiguous, rows not overlapping")
    if stream is not None or idx != _get_device():
        return _elsewhere(verify_drafts, idx, stream, (tokens, target_probs, draft_probs, uniforms, sample_u, starts), {})
    out = tokens.new_empty((rows,))
    accepted = tokens.new_empty((seqs,))
    rc = _fns()[4](tokens.data_ptr(), target_probs.data_ptr(), t0, None if draft_probs is None else draft_probs.data_ptr(),
                   d0, uniforms.data_ptr(), sample_u.data_ptr(), starts.data_ptr(), seqs, rows, vocab, out.data_ptr(),
                   accepted.data_ptr(), _status_of(idx), _raw_stream(idx))
    if rc:
        _lib.check(rc, "megakernel_verify_drafts")
    return out, accepted


def _need(ok, what: str) -> None:
    if not ok:
        raise ValueError(what)


class PagedCache8:
    """The 8-bit pools of a model's layers and one page table for all of them.

    codes [layers, pages, 2, kv_heads, page_size, head_dim], scales [layers,
    pages, 2, kv_heads].  ``reserve`` gives a sequence pages for its first n
    positions (a host-side free list; the table is copied to the device when it
    changed), ``release`` takes them back."""

    def __init__(self, layers, kv_heads, head_dim, pages, seqs, max_seq, *, page_size=64, kv_dtype="fp8", device=0):
        _need(kv_dtype in KV_DTYPES, f"kv_dtype: one of {tuple(KV_DTYPES)}")
        _need(page_size in PAGE_SIZES, f"page_size: one of {PAGE_SIZES}")
        _need(head_dim in HEAD_DIMS, f"head_dim: one of {HEAD_DIMS}")
        _need(min(layers, kv_heads, pages, seqs, max_seq) >= 1, "layers, kv_heads, pages, seqs, max_seq: at least 1")
        self.page_size, self.kv_dtype, self.max_seq = page_size, kv_dtype, max_seq
        self.device = torch.device("cuda", device)
        self.codes = torch.zeros(layers, pages, 2, kv_heads, page_size, head_dim, dtype=torch.int8,
                                 device=self.device).view(KV_DTYPES[kv_dtype])
        self.scales = torch.ones(layers, pages, 2, kv_heads, device=self.device)
        self.page_table = torch.zeros(seqs, -(-max_seq // page_size), dtype=torch.int32, device=self.device)
        self._free = list(range(pages - 1, -1, -1))
        self._held = [[] for _ in range(seqs)]

    def reserve(self, seq, positions):
        """Pages for positions [0, positions) of a sequence."""
        if positions > self.max_seq:
            _lib.check(-4, "PagedCache8.reserve")
        held, need = self._held[seq], -(-positions // self.page_size)
        if need - len(held) > len(self._free):
            _lib.check(-4, "PagedCache8.reserve")
        if need > len(held):
            begin = len(held)
            held += [self._free.pop() for _ in range(need - begin)]
            self.page_table[seq, begin:need] = torch.tensor(held[begin:], dtype=torch.int32).to(self.device)

    def release(self, seq):
        """Give a sequence's pages back."""
        self._free += reversed(self._held[seq])
        self._held[seq] = []

    def append(self, layer, k, v, starts, first, stream=None):
        kv8_append(self.codes[layer], self.scales[layer], k, v, self.page_table, starts, first, stream=stream)

    def read(self, layer, starts, first, rows, dtype=torch.bfloat16, stream=None):
        return kv8_read(self.codes[layer], self.scales[layer], self.page_table, starts, first, rows, dtype=dtype,
                        stream=stream)

    def attend(self, layer, q, starts, first, **kw):
        return kv8_attend(q, self.codes[layer], self.scales[layer], self.page_table, starts, first, **kw)
