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

import contextlib
import ctypes
import math

import torch

from . import _lib

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
FORMATS = {torch.float8_e4m3fn: 0, torch.int8: 1}
KV_DTYPES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
PAGE_SIZES = (16, 32, 64)
HEAD_DIMS = (64, 128)

_status = {}


def _status_of(device: torch.device) -> torch.Tensor:
    """The device's status word; made (and waited for) at its first use."""
    t = _status.get(device.index)
    if t is None:
        t = _status[device.index] = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()
    return t


def check(device=None) -> None:
    """Wait for the device and raise if a kernel of this module met metadata
    out of range since the last check (page ids, positions, row starts)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    t = _status_of(dev)
    torch.cuda.synchronize(dev)
    rc = int(t.item())
    if rc:
        t.zero_()
        torch.cuda.synchronize(dev)
        _lib.check(rc, "paged operators")


def _need(ok, what: str) -> None:
    if not ok:
        raise ValueError(what)


@contextlib.contextmanager
def _on(device, stream, tensors):
    """Run on `device`, on `stream` if one is given; tensors used on a stream
    that is not theirs are kept until it has passed."""
    with torch.cuda.device(device):
        if stream is None:
            yield torch.cuda.current_stream(device).cuda_stream
            return
        with torch.cuda.stream(stream):
            for t in tensors:
                if t is not None:
                    t.record_stream(stream)
            yield stream.cuda_stream


def _rows(t, name, heads_dim=True):
    """A [rows, heads, head_dim] operand whose rows can be read in 16-byte vectors."""
    _need(t.dim() == 3 and t.is_cuda, f"{name}: a CUDA tensor [rows, heads, head_dim]")
    _need(t.dtype in TYPES, f"{name}: float32, bfloat16 or float16")
    per = 16 // t.element_size()
    s = t.stride()
    one = t.shape[0] > 1
    _need((t.shape[2] <= 1 or s[2] == 1) and (not one or s[0] % per == 0) and (t.shape[1] <= 1 or s[1] % per == 0)
          and s[0] >= 0 and s[1] >= 0 and t.data_ptr() % 16 == 0,
          f"{name}: head_dim contiguous, rows and heads at multiples of 16 bytes")
    return (s[0] if one else 0, s[1] if t.shape[1] > 1 else 0)


def _int32(t, name, shape, device):
    _need(t.dtype == torch.int32 and t.device == device and tuple(t.shape) == shape and t.is_contiguous(),
          f"{name}: contiguous int32 {list(shape)} on {device}")


def _cache(codes, scales, page_table, starts, first, rows):
    _need(codes.dim() == 5 and codes.dtype in FORMATS and codes.is_cuda and codes.shape[1] == 2,
          "codes: CUDA float8_e4m3fn or int8 [pages, 2, kv_heads, page_size, head_dim]")
    pages, _, hk, page, d = codes.shape
    _need(page in PAGE_SIZES, f"page_size: one of {PAGE_SIZES}")
    _need(d in HEAD_DIMS, f"head_dim: one of {HEAD_DIMS}")
    s = codes.stride()
    _need(s[4] == 1 and s[3] == d and (hk == 1 or s[2] == page * d) and s[1] == hk * page * d,
          "codes: a page's codes contiguous")
    page_stride = s[0] if pages > 1 else 2 * hk * page * d
    _need(page_stride >= 2 * hk * page * d and page_stride % 16 == 0 and codes.data_ptr() % 16 == 0,
          "codes: pages at multiples of 16 bytes")
    dev = codes.device
    _need(scales.dtype == torch.float32 and scales.device == dev and tuple(scales.shape) == (pages, 2, hk)
          and (hk == 1 or scales.stride(2) == 1) and scales.stride(1) == hk,
          "scales: float32 [pages, 2, kv_heads], a page's scales contiguous")
    scale_stride = scales.stride(0) if pages > 1 else 2 * hk
    _need(scale_stride >= 2 * hk, "scales: pages must not overlap")
    _need(page_table.dim() == 2 and page_table.dtype == torch.int32 and page_table.device == dev
          and (page_table.shape[1] <= 1 or page_table.stride(1) == 1), "page_table: int32 [seqs, pages] on the cache's device")
    b, width = page_table.shape
    table_stride = page_table.stride(0) if b > 1 else width
    _need(table_stride >= width, "page_table: rows must not overlap")
    _int32(starts, "starts", (b + 1,), dev)
    _int32(first, "first", (b,), dev)
    return _lib.MkKv8(codes.data_ptr(), scales.data_ptr(), page_table.data_ptr(), starts.data_ptr(),
                      first.data_ptr(), page_stride, scale_stride, table_stride, pages, width, hk, page, d,
                      FORMATS[codes.dtype], b, rows)


def qk_norm_rope(q, k, q_gain, k_gain, cos, sin, positions, *, eps=1e-6, q_out=None, k_out=None, stream=None):
    """RMS norm and rotation of every head of q [rows, q_heads, D] and k
    [rows, kv_heads, D] in one pass; returns (q_out, k_out).

    q, k, the gains [D] and the outputs share a dtype; q and k may be slices
    of one packed projection, and an output may be its input.  cos, sin: fp32
    tables [positions, D / 2]; positions: int32 [rows].  D 64 or 128.  A row
    whose position is outside the tables is not written (see ``check``)."""
    dev = q.device
    qs, ks = _rows(q, "q"), _rows(k, "k")
    rows, hq, d = q.shape
    _need(k.shape[0] == rows and k.shape[2] == d and k.dtype == q.dtype and k.device == dev,
          "k: q's rows, head_dim, dtype and device")
    _need(d in HEAD_DIMS, f"head_dim: one of {HEAD_DIMS}")
    for g, name in ((q_gain, "q_gain"), (k_gain, "k_gain")):
        _need(g.dtype == q.dtype and g.device == dev and tuple(g.shape) == (d,) and g.is_contiguous()
              and g.data_ptr() % 16 == 0, f"{name}: contiguous [{d}] of q's dtype")
    _need(cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] == d // 2 and cos.dtype == sin.dtype == torch.float32
          and cos.device == dev and sin.device == dev and cos.is_contiguous() and sin.is_contiguous()
          and cos.data_ptr() % 16 == 0 and sin.data_ptr() % 16 == 0, f"cos, sin: contiguous float32 [positions, {d // 2}]")
    _int32(positions, "positions", (rows,), dev)
    _need(eps >= 0.0, "eps: not negative")
    with _on(dev, stream, (q, k, q_gain, k_gain, cos, sin, positions, q_out, k_out)) as st:
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        if k_out is None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=dev)
        qo, ko = _rows(q_out, "q_out"), _rows(k_out, "k_out")
        _need(q_out.shape == q.shape and k_out.shape == k.shape and q_out.dtype == k_out.dtype == q.dtype
              and q_out.device == k_out.device == dev, "q_out, k_out: the shapes, dtype and device of q and k")
        a = _lib.MkQkNormRope(q.data_ptr(), k.data_ptr(), q_gain.data_ptr(), k_gain.data_ptr(), q_out.data_ptr(),
                              k_out.data_ptr(), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), *qs, *ks, *qo,
                              *ko, cos.shape[0], rows, hq, k.shape[1], d, TYPES[q.dtype], eps)
        _lib.check(_lib.load().megakernel_qk_norm_rope(ctypes.byref(a), _status_of(dev).data_ptr(), st),
                   "megakernel_qk_norm_rope")
    return q_out, k_out


def kv8_append(codes, scales, k, v, page_table, starts, first, *, stream=None):
    """Quantise k and v [rows, kv_heads, D] into the cache at their rows' positions.

    A page's scale is the smallest power of two that fits the magnitudes
    written to it; a page that already holds earlier positions keeps the larger
    of its scale and the new one, its earlier codes rounded again if that grows.
    ``codes`` and ``scales`` are updated in place.  No two sequences of a call
    may write to one page."""
    ks, vs = _rows(k, "k"), _rows(v, "v")
    c = _cache(codes, scales, page_table, starts, first, k.shape[0])
    dev = codes.device
    _need(k.shape == v.shape and k.dtype == v.dtype and k.device == v.device == dev
          and k.shape[1] == c.kv_heads and k.shape[2] == c.head_dim,
          "k, v: one shape [rows, kv_heads, head_dim] and dtype, on the cache's device")
    with _on(dev, stream, (codes, scales, k, v, page_table, starts, first)) as st:
        _lib.check(_lib.load().megakernel_kv8_append(ctypes.byref(c), k.data_ptr(), *ks, v.data_ptr(), *vs,
                                                     TYPES[k.dtype], _status_of(dev).data_ptr(), st),
                   "megakernel_kv8_append")


def kv8_read(codes, scales, page_table, starts, first, rows, *, dtype=torch.bfloat16, stream=None):
    """The cached keys and values of the rows' positions: (k, v), each
    [rows, kv_heads, D] of `dtype`.  rows: starts[-1], as a number."""
    c = _cache(codes, scales, page_table, starts, first, int(rows))
    _need(rows >= 0, "rows: not negative")
    _need(dtype in TYPES, "dtype: float32, bfloat16 or float16")
    dev = codes.device
    with _on(dev, stream, (codes, scales, page_table, starts, first)) as st:
        kv = torch.empty(2, rows, c.kv_heads, c.head_dim, dtype=dtype, device=dev)
        k, v = kv[0], kv[1]
        _lib.check(_lib.load().megakernel_kv8_read(ctypes.byref(c), k.data_ptr(), v.data_ptr(), TYPES[dtype],
                                                   _status_of(dev).data_ptr(), st), "megakernel_kv8_read")
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
    qs = _rows(q, "q")
    rows, hq, d = q.shape
    c = _cache(codes, scales, page_table, starts, first, rows)
    dev = codes.device
    _need(q.dtype in (torch.bfloat16, torch.float16) and q.device == dev and d == c.head_dim,
          "q: bfloat16 or float16 [rows, q_heads, head_dim] on the cache's device")
    _need(hq >= 1 and hq % c.kv_heads == 0, "q_heads: a multiple of kv_heads")
    _need(c.seqs > 0 or rows == 0, "rows without a sequence")
    if kv_lens is not None:
        _int32(kv_lens, "kv_lens", (c.seqs,), dev)
    _need(window >= 0, "window: not negative")
    sm_scale = d ** -0.5 if sm_scale is None else float(sm_scale)
    _need(0.0 < sm_scale < math.inf, "sm_scale: positive")
    with _on(dev, stream, (q, codes, scales, page_table, starts, first, kv_lens, out)) as st:
        if out is None:
            out = torch.empty(rows, hq, d, dtype=q.dtype, device=dev)
        else:
            _need(out.shape == q.shape and out.dtype == q.dtype and out.device == dev and out.is_contiguous()
                  and out.data_ptr() % 16 == 0, "out: contiguous, of q's shape, dtype and device")
        lse = torch.empty(rows, hq, dtype=torch.float32, device=dev) if return_lse else None
        _lib.check(_lib.load().megakernel_kv8_attend(
            ctypes.byref(c), q.data_ptr(), *qs, hq, TYPES[q.dtype], sm_scale, int(bool(causal)), int(window),
            None if kv_lens is None else kv_lens.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(),
            _status_of(dev).data_ptr(), st), "megakernel_kv8_attend")
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
    _need(target_probs.dim() == 2 and target_probs.is_cuda and target_probs.dtype == torch.float32
          and (target_probs.shape[1] == 1 or target_probs.stride(1) == 1), "target_probs: CUDA float32 [rows, vocab], vocab contiguous")
    rows, vocab = target_probs.shape
    dev = target_probs.device
    _need(vocab >= 1, "vocab: at least one token")
    _need(starts.dim() == 1 and starts.shape[0] >= 1, "starts: int32 [seqs + 1]")
    seqs = starts.shape[0] - 1
    _int32(starts, "starts", (seqs + 1,), dev)
    _int32(tokens, "tokens", (rows,), dev)
    for t, name, n in ((uniforms, "uniforms", rows), (sample_u, "sample_u", seqs)):
        _need(t.dtype == torch.float32 and t.device == dev and tuple(t.shape) == (n,) and t.is_contiguous(),
              f"{name}: contiguous float32 [{n}] on {dev}")
    if draft_probs is not None:
        _need(draft_probs.shape == target_probs.shape and draft_probs.dtype == torch.float32
              and draft_probs.device == dev and (vocab == 1 or draft_probs.stride(1) == 1),
              "draft_probs: as target_probs")
    stride = [vocab if t is None or rows <= 1 else t.stride(0) for t in (target_probs, draft_probs)]
    _need(min(stride) >= vocab, "probabilities: rows must not overlap")
    with _on(dev, stream, (tokens, target_probs, draft_probs, uniforms, sample_u, starts)) as st:
        out = torch.empty(rows, dtype=torch.int32, device=dev)
        accepted = torch.empty(seqs, dtype=torch.int32, device=dev)
        _lib.check(_lib.load().megakernel_verify_drafts(
            tokens.data_ptr(), target_probs.data_ptr(), stride[0],
            None if draft_probs is None else draft_probs.data_ptr(), stride[1], uniforms.data_ptr(),
            sample_u.data_ptr(), starts.data_ptr(), seqs, rows, vocab, out.data_ptr(), accepted.data_ptr(),
            _status_of(dev).data_ptr(), st), "megakernel_verify_drafts")
    return out, accepted


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
