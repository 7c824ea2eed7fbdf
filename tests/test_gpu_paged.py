"""The paged 8-bit serving operators against plain 64-bit models.

Tolerances, derived before the first run (u = 2^-8 for bf16, 2^-11 for f16,
2^-24 for fp32: half a unit in the last place, relative):

- norm + rotation: u |o| for the store, and 24 roundings of 2^-24 of the
  normalised halves for the fp32 arithmetic (16 squares and their sum count
  half through the square root, then root, division, gain, rotation);
- the cache holds power-of-two scales, so codes, scales and values read back
  are equal;
- attention: u |o| for the store; weights enter the second product in 11 bits,
  2^-11 of sum p |v| with the running rescaling; scores carry at most 2^-20 of
  sum |q k| from the fp32 accumulation, which moves each weight and the sum by
  that much: 2 x 2^-20 x max sum |q k| x sum p |v|;
- lse: 2^-20 of max sum |q k|, and 2^-20 of |lse| + 1 for exp2, sum and log2;
- verification is in whole numbers: equal.
"""
import numpy as np
import pytest
import torch

from megakernel_b200 import paged

from . import _paged as M

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}   # half the smallest f16 step
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def starts_of(rows):
    return [0] + [int(x) for x in np.cumsum(rows)]


# ---- norm and rotation -----------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,hq,hk,layout", [(1, 16, 8, "packed"), (0, 2, 1, "plain"), (3, 1, 1, "plain"),
                                               (65, 4, 2, "packed"), (513, 5, 3, "heads_first"), (7, 16, 8, "inplace")])
def test_norm_rope(dtype, d, rows, hq, hk, layout):
    g = torch.Generator().manual_seed(rows * 31 + hq + d)
    x = torch.randn(rows, hq + 2 * hk, d, generator=g).to(dtype).to(DEV)
    if rows:
        x[0, 0] = 0                       # a head of zeros: eps alone
        x[-1, -2 * hk] *= 2.0 ** -12      # small against eps
    if layout == "heads_first":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    q, k = x[:, :hq], x[:, hq:hq + hk]
    if layout == "plain":
        q, k = q.contiguous(), k.contiguous()
    qg, kg = ((1 + 0.3 * torch.randn(d, generator=g)).to(dtype).to(DEV) for _ in range(2))
    table = 777
    ang = torch.arange(table)[:, None] * 1e6 ** (-torch.arange(0, d, 2) / d)
    cos, sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    pos = torch.randint(0, table, (rows,), generator=g, dtype=torch.int32).to(DEV)
    if rows:
        pos[-1] = table - 1
    want = []
    for t, gain in ((q, qg), (k, kg)):
        t, gain = t.cpu().double(), gain.cpu().double()
        y = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * gain
        y1, y2 = y.chunk(2, -1)
        c, s = (v.cpu().double()[pos.cpu().long()][:, None] for v in (cos, sin))
        o = torch.cat([y1 * c - y2 * s, y2 * c + y1 * s], -1)
        want.append((o, (y1.abs() + y2.abs()).repeat(1, 1, 2)))
    kw = dict(q_out=q, k_out=k) if layout == "inplace" else {}
    got = paged.qk_norm_rope(q, k, qg, kg, cos, sin, pos, eps=1e-6, **kw)
    paged.check(DEV)
    for o, (ref, mag) in zip(got, want):
        err = (o.cpu().double() - ref).abs()
        assert (err <= U[dtype] * ref.abs() + 24 * 2.0 ** -24 * mag + TINY[dtype]).all(), err.max()


def test_norm_rope_position_outside_tables_is_reported():
    q, k = torch.ones(3, 2, 64, device=DEV), torch.ones(3, 1, 64, device=DEV)
    cos = sin = torch.ones(5, 32, device=DEV)
    one = torch.ones(64, device=DEV)
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    paged.qk_norm_rope(q, k, one, one, cos, sin, ints([4, 5, -1]), q_out=qo, k_out=ko)
    with pytest.raises(RuntimeError):
        paged.check(DEV)
    assert (qo[1:] == 7).all() and (ko[1:] == 7).all() and not (qo[0] == 7).any()
    paged.check(DEV)   # reported once


# ---- cache write and read -----------------------------------------------------------

def pool(fmt, pages, hk, page, d, seed=0):
    """Codes and scales as leftovers of earlier use: any byte, any power of two."""
    r = np.random.RandomState(seed)
    codes = r.randint(0, 256, (pages, 2, hk, page, d)).astype(np.uint8)
    scales = 2.0 ** r.randint(-8, 9, (pages, 2, hk))
    c = torch.from_numpy(codes.view(np.int8)).to(DEV).view(M.DT[fmt])
    return codes, scales, c, torch.from_numpy(scales).float().to(DEV)


def table_for(lens, page, seed=1, spare=0):
    need = [max(1, -(-n // page)) + spare for n in lens]
    width = max(need)
    ids = np.random.RandomState(seed).permutation(len(lens) * width).reshape(len(lens), width).astype(np.int32)
    return ids, len(lens) * width


def same_codes(got, want, fmt):
    got = got.view(torch.int8).cpu().numpy().view(np.uint8)
    if fmt == "fp8":   # any NaN code is NaN
        got, want = np.where(got & 127 == 127, 127, got), np.where(want & 127 == 127, 127, want)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("dtype,page,d,hk", [(BF, 16, 64, 2), (HF, 32, 128, 1), (FP, 64, 64, 3), (BF, 64, 128, 2),
                                             (FP, 16, 128, 1), (HF, 64, 64, 1)])
def test_append_calls_in_a_row_and_read(fmt, dtype, page, d, hk):
    """Prompts, then single tokens that grow, keep and cross pages; codes, scales and read-back."""
    r = np.random.RandomState(page + d + hk)
    rounds = [([5, page + 3, 0, 2 * page, 1], [0, 0, 0, 0, page - 1])]
    for _ in range(4):
        rows, first = rounds[-1]
        rounds.append(([1, 2, 1, 1, 1], [f + n for f, n in zip(first, rows)]))
    lens = [f + n for f, n in zip(*reversed(rounds[-1]))]
    ids, pages = table_for(lens, page)
    codes, scales, dc, ds = pool(fmt, pages, hk, page, d)
    # the page in front of sequence 4's first row holds real codes
    codes[ids[4][0]] &= 0x3F
    dc.view(torch.int8)[int(ids[4][0])] &= 0x3F
    model = M.Model(codes, scales, fmt)
    table = ints(ids.tolist())
    for i, (rows, first) in enumerate(rounds):
        st, size = starts_of(rows), 4.0 ** i if i < 3 else 0.01
        k, v = (torch.from_numpy(r.standard_normal((st[-1], hk, d)) * size).to(dtype) for _ in range(2))
        if i == 1:   # an outlier, infinities, NaN, a row of zeros
            k[0, 0, 3], k[1, 0, 5], v[0, 0, 1], v[2, 0] = 300.0, float("inf"), float("nan"), 0.0
            v[1, 0, 2] = float("-inf")
        model.append(k.float().numpy(), v.float().numpy(), ids, st, first)
        paged.kv8_append(dc, ds, k.to(DEV), v.to(DEV), table, ints(st), ints(first))
        paged.check(DEV)
        assert np.array_equal(ds.cpu().double().numpy(), model.s)
        same_codes(dc, model.c, fmt)
    st, first = starts_of([n - (b == 1) for b, n in enumerate(lens)]), [0, 1, 0, 0, 0]
    k, v = paged.kv8_read(dc, ds, table, ints(st), ints(first), st[-1], dtype=dtype)
    for b in range(5):
        x = M.values(dc, ds, ids[b], lens[b], fmt)[first[b]:]
        for got, kv in ((k, 0), (v, 1)):
            want = x[:, kv].to(dtype)
            assert torch.equal(torch.nan_to_num(got[st[b]:st[b + 1]].cpu()), torch.nan_to_num(want)), (b, kv)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_append_padding_strides_and_pool_strides(fmt):
    """Negative positions are skipped; k and v slices of a packed projection; a layer's slice of a pool of layers."""
    page, d, hk, layers = 16, 64, 2, 3
    rows, first = [6, 3, 4], [-2, -3, 7]
    st = starts_of(rows)
    x = torch.randn(st[-1], 4 + 2 * hk, d, generator=torch.Generator().manual_seed(3)).to(BF).to(DEV)
    k, v = x[:, 4:4 + hk], x[:, 4 + hk:]
    codes = torch.zeros(8, layers, 2, hk, page, d, dtype=torch.int8, device=DEV)
    scales = torch.ones(8, layers, 2, hk, device=DEV)
    ids = [[5], [0], [3]]
    dc, ds = codes[:, 1].view(M.DT[fmt]) if fmt == "int8" else codes.view(M.DT[fmt])[:, 1], scales[:, 1]
    model = M.Model(codes[:, 1].cpu().numpy().view(np.uint8), ds.cpu().numpy(), fmt)
    model.append(k.float().cpu().numpy(), v.float().cpu().numpy(), ids, st, first)
    paged.kv8_append(dc, ds, k, v, ints(ids), ints(st), ints(first))
    paged.check(DEV)
    same_codes(codes[:, 1], model.c, fmt)
    assert np.array_equal(ds.cpu().double().numpy(), model.s)
    assert not codes[:, 0].any() and not codes[:, 2].any() and (scales[:, 0] == 1).all()


def test_append_and_read_report_bad_metadata_and_touch_nothing_else():
    page, d, hk = 16, 64, 1
    dc = torch.zeros(4, 2, hk, page, d, dtype=torch.int8, device=DEV)
    ds = torch.ones(4, 2, hk, device=DEV)
    k = torch.ones(2, hk, d, device=DEV)
    for table, first in (([[4]], [0]), ([[-1]], [0]), ([[0]], [15]), ([[0]], [1 << 20])):
        paged.kv8_append(dc, ds, k, k, ints(table), ints([0, 2]), ints(first))
        with pytest.raises(RuntimeError):
            paged.check(DEV)
        paged.kv8_read(dc, ds, ints(table), ints([0, 2]), ints(first), 2)
        with pytest.raises(RuntimeError):
            paged.check(DEV)
    for starts in ([0, 3], [-1, 1], [2, 0]):
        before = dc.clone()
        paged.kv8_append(dc, ds, k, k, ints([[2]]), ints(starts), ints([0]))
        with pytest.raises(RuntimeError):
            paged.check(DEV)
        assert torch.equal(before, dc)
    assert not dc[2:].any()


# ---- attention ---------------------------------------------------------------------

def attend_case(fmt, dtype, page, d, hq, hk, rows, lens, seed=0, general=False, **kw):
    """Random caches (leftovers beyond each length: NaN codes or the lowest int8, huge scales), against 64 bits."""
    g = torch.Generator().manual_seed(seed + 7 * page + d + hq + sum(rows))
    st = starts_of(rows)
    first = kw.pop("first", None) or [n - r for n, r in zip(lens, rows)]
    kvl = kw.pop("kv_lens", None)
    held = kvl if kvl is not None else lens
    ids, pages = table_for([max(1, n) for n in held], page, spare=1)
    codes = torch.full((pages, 2, hk, page, d), 0x7F if fmt == "fp8" else -128, dtype=torch.int8)
    scales = torch.full((pages, 2, hk), 2.0 ** 30)
    for b, n in enumerate(held):
        for j in range(-(-max(n, 0) // page)):
            fill = min(page, n - j * page)
            x = torch.randn(2, hk, fill, d, generator=g)
            if fmt == "fp8":
                c = (x * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.int8)
            else:
                c = (x * 30).round().clamp(-127, 127).to(torch.int8)
            codes[ids[b][j], :, :, :fill] = c
            unit = 0.01 if fmt == "fp8" else 0.03
            sc = unit * (1 + torch.rand(2, hk, generator=g)) if general else \
                2.0 ** torch.randint(-7, -4, (2, hk), generator=g).float()
            scales[ids[b][j]] = sc
    q = (1.5 * torch.randn(st[-1], hq, d, generator=g)).to(dtype)
    kvs = [M.values(codes.view(M.DT[fmt]), scales, ids[b], max(n, 0), fmt) for b, n in enumerate(held)]
    want, wl, mag, dots = M.attend(q, kvs, st, first, kv_lens=kvl, **kw)
    out, lse = paged.kv8_attend(q.to(DEV), codes.to(DEV).view(M.DT[fmt]), scales.to(DEV), ints(ids.tolist()), ints(st),
                                ints(first), kv_lens=None if kvl is None else ints(kvl), return_lse=True, **kw)
    paged.check(DEV)
    out, lse = out.cpu().double(), lse.cpu().double()
    tol = U[dtype] * want.abs() + (2.0 ** -11 + 2 * 2.0 ** -20 * dots[..., None]) * mag + TINY[dtype]
    bad = ~((out - want).abs() <= tol)
    assert not bad.any(), ((out - want).abs() / tol.clamp(min=1e-30)).nan_to_num(1e9).max()
    empty = torch.isinf(wl)
    assert torch.equal(torch.isinf(lse), empty) and (out[empty] == 0).all()
    ltol = 2.0 ** -20 * (dots + wl.abs() + 1)
    assert ((lse - wl).abs()[~empty] <= ltol[~empty]).all(), ((lse - wl).abs() / ltol)[~empty].max()


LENS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("fmt,dtype", [("fp8", BF), ("int8", HF)])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(4, 2), (3, 3), (8, 1)])
def test_attend_single_rows_at_all_lengths(fmt, dtype, page, d, hq, hk):
    attend_case(fmt, dtype, page, d, hq, hk, [1] * len(LENS), LENS)


@pytest.mark.parametrize("fmt,dtype", [("fp8", HF), ("int8", BF)])
@pytest.mark.parametrize("page,d,hq,hk", [(16, 64, 16, 8), (64, 128, 4, 2), (32, 64, 5, 1), (64, 64, 2, 2),
                                          (16, 128, 7, 1)])
def test_attend_drafts(fmt, dtype, page, d, hq, hk):
    """A few rows per sequence, causal among themselves; one sequence has none."""
    attend_case(fmt, dtype, page, d, hq, hk, [3, 1, 0, 8, 5, 2], [3, 70, 40, 129, 1100, 2])


@pytest.mark.parametrize("fmt,dtype", [("fp8", BF), ("int8", HF)])
@pytest.mark.parametrize("page,d,hq,hk", [(16, 64, 4, 2), (64, 128, 4, 2), (32, 128, 3, 1), (64, 64, 2, 2)])
@pytest.mark.parametrize("rows,lens", [([129], [129]), ([64, 200], [64, 333]), ([1, 257, 17], [90, 500, 17])])
def test_attend_prompts(fmt, dtype, page, d, hq, hk, rows, lens):
    attend_case(fmt, dtype, page, d, hq, hk, rows, lens)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("window", [1, 2, 16, 63, 100])
@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [5, 64, 700]), ([150, 3], [400, 99])])
def test_attend_window(fmt, window, rows, lens):
    attend_case(fmt, BF, 32, 64, 4, 2, rows, lens, window=window)


@pytest.mark.parametrize("rows,lens", [([2, 1, 3, 2], None), ([130, 1, 70, 2], None)])
def test_attend_empty_rows(rows, lens):
    """kv_lens of zero, padding rows at negative positions, and a window past the end see nothing."""
    first = [0, 10, -2, 500]
    attend_case("fp8", BF, 16, 64, 4, 2, rows, None, first=first, kv_lens=[0, 7, 90, 100], window=64)
    attend_case("int8", HF, 64, 128, 4, 2, rows, None, first=first, kv_lens=[0, 0, 1, 100])


@pytest.mark.parametrize("rows", [[1, 4, 2], [140, 65, 1]])
def test_attend_without_causal_mask(rows):
    attend_case("fp8", BF, 32, 128, 4, 2, rows, None, first=[3, 0, 600], kv_lens=[77, 200, 0], causal=False)
    attend_case("int8", BF, 16, 64, 2, 1, rows, [400, 200, 9], causal=False, sm_scale=0.31)


def test_attend_general_scales_and_large_scores():
    """Scales that are no powers of two; scores of some hundreds."""
    attend_case("fp8", BF, 32, 64, 4, 2, [1, 3], [500, 77], general=True)
    attend_case("int8", HF, 64, 128, 4, 2, [1, 3, 140], [500, 77, 300], general=True, sm_scale=2.0)


def test_attend_long_context_few_rows():
    attend_case("fp8", BF, 64, 64, 16, 8, [1], [8192])
    attend_case("int8", HF, 16, 64, 4, 2, [2], [20001])


def test_attend_strided_queries_other_stream_and_repeat():
    """q as a slice of a packed projection, on a side stream; two calls give the same bits."""
    g = torch.Generator().manual_seed(5)
    page, d, hq, hk, n = 32, 64, 4, 2, 2000
    pages = -(-n // page)
    codes = torch.randn(pages, 2, hk, page, d, generator=g).mul(100).to(torch.float8_e4m3fn).to(DEV)
    scales = torch.full((pages, 2, hk), 2.0 ** -6, device=DEV)
    x = torch.randn(5, hq + 2 * hk, d, generator=g).to(BF).to(DEV)
    args = (codes, scales, ints([list(range(pages))]), ints([0, 5]), ints([n - 5]))
    a = paged.kv8_attend(x[:, :hq], *args)
    b = paged.kv8_attend(x[:, :hq].contiguous(), *args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c = paged.kv8_attend(x[:, :hq], *args, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    a, b, c = (t.view(torch.int16) for t in (a, b, c))   # bits: a few codes of the cache are NaN
    assert torch.equal(a, b) and torch.equal(a, c)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes whose used pages lie at its end."""
    page, d, hk = 64, 128, 8
    pages = (1 << 32) // (2 * hk * page * d) + 40
    codes = torch.empty(pages, 2, hk, page, d, dtype=torch.int8, device=DEV).view(torch.float8_e4m3fn)
    scales = torch.ones(pages, 2, hk, device=DEV)
    n = 150
    table = [[pages - 1, pages - 3, pages - 2]]
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(n, hk, d, generator=g).to(BF).to(DEV) for _ in range(2))
    paged.kv8_append(codes, scales, k, v, ints(table), ints([0, n]), ints([0]))
    k2, v2 = paged.kv8_read(codes, scales, ints(table), ints([0, n]), ints([0]), n)
    paged.check(DEV)
    # e4m3 keeps 3 bits after the leading one: 2^-4 relative, or half a subnormal step of a page's scale
    for x, y in ((k, k2), (v, v2)):
        assert ((x.float() - y.float()).abs() <= 2.0 ** -4 * x.float().abs() + 2.0 ** -10 * 2.0 ** -6).all()
    q = torch.randn(2, 16, d, generator=g).to(BF)
    kv = torch.stack([k2, v2], 1).cpu().double()
    want, _, mag, dots = M.attend(q, [kv], [0, 2], [n - 2])
    out = paged.kv8_attend(q.to(DEV), codes, scales, ints(table), ints([0, 2]), ints([n - 2]))
    paged.check(DEV)
    tol = U[BF] * want.abs() + (2.0 ** -11 + 2 * 2.0 ** -20 * dots[..., None]) * mag
    assert ((out.cpu().double() - want).abs() <= tol).all()


def test_attend_reports_bad_pages():
    page, d = 16, 64
    codes = torch.zeros(2, 2, 1, page, d, dtype=torch.int8, device=DEV)
    scales = torch.ones(2, 2, 1, device=DEV)
    for rows in (1, 200):
        q = torch.ones(rows, 1, d, device=DEV, dtype=BF)
        for table, first in (([[0, 9]], [20]), ([[0, 1]], [400]), ([[-5, 0]], [3])):
            paged.kv8_attend(q, codes, scales, ints(table), ints([0, rows]), ints(first))
            with pytest.raises(RuntimeError):
                paged.check(DEV)


# ---- verification ---------------------------------------------------------------------

def probs(r, rows, vocab, sharp=2.0):
    x = r.standard_normal((rows, vocab)) * sharp
    e = np.exp(x - x.max(1, keepdims=True))
    return (e / e.sum(1, keepdims=True)).astype(np.float32)


def verify_case(tokens, target, draft, u, su, st, strided=False):
    want, wacc = M.verify(tokens, target, draft, u, su, st)

    def dev(p):
        if p is None:
            return None
        t = torch.from_numpy(p)
        if strided:
            wide = torch.full((t.shape[0], t.shape[1] + 5), 9.0)
            wide[:, :t.shape[1]] = t
            return wide.to(DEV)[:, :t.shape[1]]
        return t.to(DEV)

    out, acc = paged.verify_drafts(ints(list(tokens)), dev(target), dev(draft), torch.tensor(u, dtype=FP, device=DEV),
                                   torch.tensor(su, dtype=FP, device=DEV), ints(st))
    paged.check(DEV)
    assert acc.cpu().tolist() == wacc
    assert out.cpu().tolist() == want


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 1000, 2048, 4097, 151936])
@pytest.mark.parametrize("with_draft", [True, False])
def test_verify(vocab, with_draft):
    r = np.random.RandomState(vocab + with_draft)
    rows = [1, 4, 0, 8, 2, 5, 3]
    st = starts_of(rows)
    target = probs(r, st[-1], vocab)
    draft = np.where(r.rand(st[-1], 1) < 0.5, target, probs(r, st[-1], vocab)).astype(np.float32)
    tokens = [int(np.argmax(draft[t - 1])) if r.rand() < 0.7 else r.randint(vocab) for t in range(st[-1])]
    u, su = r.rand(st[-1]).astype(np.float32), r.rand(len(rows)).astype(np.float32)
    verify_case(tokens, target, draft if with_draft else None, u, su, st, strided=vocab < 5000)


def test_verify_edges():
    """Random numbers at 0 and just under 1; rows of zeros, NaN and values over 1; equal distributions; drafts
    outside the vocabulary; a draft with no probability on either side."""
    r = np.random.RandomState(2)
    v, n = 37, 3
    top = np.float32(1 - 2.0 ** -24)
    for u0 in (0.0, top):
        for s0 in (0.0, top):
            target, draft = probs(r, 6 * n, v), probs(r, 6 * n, v)
            draft[0:n] = target[0:n]                         # never refused
            target[n] = 0                                    # nothing to keep or draw
            target[2 * n, ::2] = np.nan
            target[3 * n, 5] = 3.0
            draft[3 * n, 5] = np.inf
            tokens = r.randint(0, v, 6 * n)
            tokens[3 * n + 1], tokens[4 * n + 1], tokens[5 * n + 1] = 5, v, -1
            target[4 * n + 1, tokens[4 * n + 2]] = draft[4 * n + 1, tokens[4 * n + 2]] = 0
            u, su = np.full(6 * n, u0, np.float32), np.full(6, s0, np.float32)
            for d in (draft, None):
                verify_case(tokens.tolist(), target, d, u, su, list(range(0, 6 * n + 1, n)))


def test_verify_last_tokens_of_the_vocabulary():
    """All weight on the first or the last token, at sizes around a thread's share."""
    for v in (1023, 1024, 1025, 2049, 50257):
        for at in (0, v - 1):
            target = np.zeros((2, v), np.float32)
            target[:, at] = 1
            verify_case([3 % v, at], target, None, np.array([0.5, 0.5], np.float32), np.array([0.999], np.float32), [0, 2])


def test_verify_many_drafts_and_sequences():
    r = np.random.RandomState(4)
    rows = [40] + [2] * 300 + [1100]
    st = starts_of(rows)
    target = probs(r, st[-1], 50, 0.3)
    tokens = r.randint(0, 50, st[-1]).tolist()
    u = (r.rand(st[-1]) * 0.01).astype(np.float32)
    verify_case(tokens, target, target.copy(), u, r.rand(len(rows)).astype(np.float32), st)


@pytest.mark.parametrize("rows", [3, 150])
def test_attend_nan_in_places_that_only_some_rows_see(rows):
    """A NaN value code counts for the rows that see its position, and for them only."""
    page, d, hq, hk, n = 16, 64, 2, 1, rows + 21
    pages = -(-n // page)
    g = torch.Generator().manual_seed(rows)
    codes = torch.randn(pages, 2, hk, page, d, generator=g).clamp(-4, 4).mul(100).to(torch.float8_e4m3fn).view(torch.int8)
    marks = [(n - 1, 5), (n - 2, 63), (n - rows + 1, 0)]
    for pos, dim in marks:
        codes[pos // page, 1, 0, pos % page, dim] = -1          # 0xff
    q = torch.randn(rows, hq, d, generator=g).to(BF).to(DEV)
    out = paged.kv8_attend(q, codes.to(DEV).view(torch.float8_e4m3fn), torch.full((pages, 2, hk), 2.0 ** -6, device=DEV),
                           ints([list(range(pages))]), ints([0, rows]), ints([n - rows]))
    paged.check(DEV)
    want = torch.zeros(rows, d, dtype=torch.bool)
    for pos, dim in marks:
        want[max(0, pos - (n - rows)):, dim] = True
    assert torch.equal(out.isnan().cpu(), want[:, None].expand(rows, hq, d))


@pytest.mark.parametrize("seqs,hq,hk,rows,length", [(70, 4, 2, 1, 90), (150, 2, 1, 2, 200), (330, 8, 8, 1, 40), (100, 4, 4, 30, 60)])
def test_attend_many_sequences(seqs, hq, hk, rows, length):
    """More sequences than a warp looks over at once, and more items than warps."""
    r = np.random.RandomState(seqs)
    n = [int(x) for x in r.randint(0, rows + 1, seqs)]
    lens = [k + int(x) for k, x in zip(n, r.randint(0, length, seqs))]
    attend_case("fp8", BF, 16, 64, hq, hk, n, lens)
