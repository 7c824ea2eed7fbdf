"""What the paged 8-bit operators refuse before anything is launched."""
import ctypes

import pytest
import torch

from megakernel_b200 import _lib, paged

from ._common import lib

FAKE = 1 << 20   # a non-null, aligned address; every call below returns before using it


def kv8(**kw):
    a = dict(codes=FAKE, scales=FAKE, page_table=FAKE, starts=FAKE, first=FAKE, page_stride=2 * 2 * 16 * 64,
             scale_stride=4, table_stride=3, num_pages=5, table_width=3, kv_heads=2, page_size=16, head_dim=64,
             format=0, seqs=1, rows=4)
    a.update(kw)
    return ctypes.byref(_lib.MkKv8(**a))


BAD_CACHES = [dict(codes=None), dict(codes=FAKE + 8), dict(scales=None), dict(page_table=None), dict(starts=None),
              dict(first=None), dict(page_stride=100), dict(page_stride=2 * 2 * 16 * 64 + 8), dict(scale_stride=3),
              dict(table_stride=2), dict(num_pages=-1), dict(table_width=-1), dict(kv_heads=0), dict(page_size=24),
              dict(page_size=128), dict(head_dim=96), dict(format=2), dict(format=-1), dict(seqs=-1), dict(rows=-1),
              dict(rows=1 << 30)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda b: "-".join(f"{k}={v}" for k, v in b.items()))
def test_c_entries_refuse_bad_caches(bad):
    L = lib()
    assert L.megakernel_kv8_append(kv8(**bad), FAKE, 128, 64, FAKE, 128, 64, 1, None, None) == -1
    assert L.megakernel_kv8_read(kv8(**bad), FAKE, FAKE, 1, None, None) == -1
    assert L.megakernel_kv8_attend(kv8(**bad), FAKE, 256, 64, 4, 1, 0.125, 1, 0, None, FAKE, None, FAKE, 1 << 30, None, None) == -1
    assert L.megakernel_kv8_attend_workspace(kv8(**bad), 4) == -1 or set(bad) & {"codes", "scales", "page_table", "starts", "first"}


def test_c_entries_refuse_bad_operands():
    L = lib()
    app, read, att = L.megakernel_kv8_append, L.megakernel_kv8_read, L.megakernel_kv8_attend
    assert app(None, FAKE, 128, 64, FAKE, 128, 64, 1, None, None) == -1
    assert app(kv8(), None, 128, 64, FAKE, 128, 64, 1, None, None) == -1
    assert app(kv8(), FAKE, 128, 64, FAKE + 4, 128, 64, 1, None, None) == -1
    assert app(kv8(), FAKE, 129, 64, FAKE, 128, 64, 1, None, None) == -1
    assert app(kv8(), FAKE, 128, 64, FAKE, 128, -64, 1, None, None) == -1
    assert app(kv8(), FAKE, 128, 64, FAKE, 128, 64, 3, None, None) == -1
    assert read(kv8(), FAKE, None, 1, None, None) == -1
    assert read(kv8(), FAKE, FAKE + 2, 1, None, None) == -1
    assert read(kv8(), FAKE, FAKE, -1, None, None) == -1

    def attend(q=FAKE, row=256, head=64, hq=4, type=1, scale=0.125, window=0, out=FAKE, work=FAKE, size=1 << 30):
        return att(kv8(), q, row, head, hq, type, scale, 1, window, None, out, None, work, size, None, None)

    for bad in (dict(q=None), dict(q=FAKE + 2), dict(row=255), dict(head=60), dict(hq=3), dict(hq=0), dict(type=0),
                dict(type=7), dict(scale=0.0), dict(scale=float("nan")), dict(window=-1), dict(out=None),
                dict(out=FAKE + 8), dict(work=None), dict(size=-1)):
        assert attend(**bad) == -1, bad


def test_c_norm_rope_refuses():
    L = lib()
    good = dict(q=FAKE, k=FAKE, q_gain=FAKE, k_gain=FAKE, q_out=FAKE, k_out=FAKE, cos=FAKE, sin=FAKE, positions=FAKE,
                q_row=256, q_head=64, k_row=128, k_head=64, qo_row=256, qo_head=64, ko_row=128, ko_head=64,
                table_rows=9, rows=3, q_heads=4, kv_heads=2, head_dim=64, type=1, eps=1e-6)
    for bad in (dict(q=None), dict(k=FAKE + 2), dict(q_gain=None), dict(k_out=None), dict(cos=None), dict(sin=None),
                dict(positions=None), dict(q_row=255), dict(ko_head=-64), dict(rows=-1), dict(q_heads=-1),
                dict(head_dim=80), dict(type=3), dict(eps=-1.0), dict(eps=float("nan")), dict(table_rows=-1)):
        a = _lib.MkQkNormRope(**{**good, **bad})
        assert L.megakernel_qk_norm_rope(ctypes.byref(a), None, None) == -1, bad
    assert L.megakernel_qk_norm_rope(None, None, None) == -1


def test_c_verify_refuses():
    L = lib()

    def verify(tokens=FAKE, target=FAKE, trow=100, draft=FAKE, drow=100, u=FAKE, su=FAKE, starts=FAKE, seqs=2, rows=5,
               vocab=100, out=FAKE, acc=FAKE):
        return L.megakernel_verify_drafts(tokens, target, trow, draft, drow, u, su, starts, seqs, rows, vocab, out, acc,
                                          None, None)

    for bad in (dict(tokens=None), dict(target=None), dict(trow=99), dict(drow=99), dict(u=None), dict(su=None),
                dict(starts=None), dict(seqs=-1), dict(rows=-1), dict(vocab=0), dict(out=None), dict(acc=None)):
        assert verify(**bad) == -1, bad


def test_empty_calls_do_nothing():
    L = lib()
    for none in (dict(rows=0), dict(seqs=0)):
        c = kv8(codes=None, scales=None, page_table=None, starts=None, first=None, **none)
        assert L.megakernel_kv8_append(c, None, 0, 0, None, 0, 0, 1, None, None) == 0
        assert L.megakernel_kv8_read(c, None, None, 1, None, None) == 0
    assert L.megakernel_kv8_attend(kv8(rows=0), None, 0, 0, 4, 1, 0.1, 1, 0, None, None, None, None, 0, None, None) == 0
    # rows that belong to no sequence
    assert L.megakernel_kv8_attend(kv8(seqs=0), FAKE, 256, 64, 4, 1, 0.1, 1, 0, None, FAKE, None, FAKE, 1 << 30, None, None) == -1
    assert L.megakernel_verify_drafts(None, None, 5, None, 5, None, None, None, 0, 0, 5, None, None, None, None) == 0


def test_python_entries_refuse_host_tensors_and_wrong_types():
    x = torch.zeros(2, 2, 64)
    i = torch.zeros(2, dtype=torch.int32)
    codes, scales = torch.zeros(3, 2, 2, 16, 64, dtype=torch.int8), torch.ones(3, 2, 2)
    table = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged.qk_norm_rope(x, x, x[0, 0], x[0, 0], x[0], x[0], i)
    with pytest.raises(ValueError):
        paged.kv8_append(codes, scales, x, x, table, i, i[:1])
    with pytest.raises(ValueError):
        paged.kv8_read(codes, scales, table, i, i[:1], 2)
    with pytest.raises(ValueError):
        paged.kv8_attend(x, codes, scales, table, i, i[:1])
    with pytest.raises(ValueError):
        paged.verify_drafts(i, torch.rand(2, 5), None, torch.rand(2), torch.rand(1), i)


def test_cache_class_refuses():
    for bad in (dict(kv_dtype="bf16"), dict(page_size=20), dict(head_dim=80), dict(pages=0), dict(seqs=0)):
        kw = dict(layers=1, kv_heads=2, head_dim=64, pages=4, seqs=1, max_seq=64)
        kw.update({k: v for k, v in bad.items() if k in kw})
        opt = {k: v for k, v in bad.items() if k not in kw}
        with pytest.raises(ValueError):
            paged.PagedCache8(**kw, **opt)


@pytest.mark.gpu
def test_python_entries_refuse_on_the_device():
    dev = torch.device("cuda", 0)
    hk, d, page = 2, 64, 16
    codes = torch.zeros(3, 2, hk, page, d, dtype=torch.int8, device=dev)
    scales = torch.ones(3, 2, hk, device=dev)
    table, starts, first = (torch.zeros(s, dtype=torch.int32, device=dev) for s in ((1, 2), (2,), (1,)))
    k = torch.zeros(2, hk, d, device=dev, dtype=torch.bfloat16)
    q = torch.zeros(2, 4, d, device=dev, dtype=torch.bfloat16)

    def append(**kw):
        a = dict(codes=codes, scales=scales, k=k, v=k, page_table=table, starts=starts, first=first)
        a.update(kw)
        paged.kv8_append(**a)

    def attend(q=q, **kw):
        opt = {n: kw.pop(n) for n in list(kw) if n in ("kv_lens", "window", "sm_scale", "out")}
        a = dict(codes=codes, scales=scales, page_table=table, starts=starts, first=first)
        a.update(kw)
        return paged.kv8_attend(q, **a, **opt)

    wide = torch.zeros(3, 2, hk, page, 2 * d, dtype=torch.int8, device=dev)
    caches = [dict(codes=codes.view(torch.uint8)), dict(codes=wide[..., :d]), dict(codes=codes[:, :1]),
              dict(codes=codes.transpose(2, 3)), dict(scales=scales.double()), dict(scales=scales[:2]),
              dict(scales=scales.cpu()), dict(page_table=table.long()), dict(page_table=table[0]),
              dict(starts=starts[:1]), dict(starts=starts.long()), dict(first=starts), dict(first=first.cpu()),
              dict(codes=torch.zeros(3, 2, hk, 8, d, dtype=torch.int8, device=dev)),
              dict(codes=torch.zeros(3, 2, hk, page, 32, dtype=torch.int8, device=dev))]
    for bad in caches:
        for call in (append, attend):
            with pytest.raises(ValueError):
                call(**bad)
    odd = torch.zeros(2, hk, d + 1, device=dev, dtype=torch.bfloat16)
    for bad in (dict(k=k.double()), dict(v=k.float()), dict(k=k[:, :1]), dict(k=odd[..., :d], v=odd[..., :d]),
                dict(k=k[..., ::2], v=k[..., ::2])):
        with pytest.raises(ValueError):
            append(**bad)
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=torch.zeros(2, 4, 128, device=dev, dtype=torch.bfloat16)),
                dict(kv_lens=starts), dict(window=-1), dict(sm_scale=0.0), dict(sm_scale=-1.0), dict(out=q.float()),
                dict(out=q[:1])):
        with pytest.raises(ValueError):
            attend(**bad)
    p = torch.rand(2, 7, device=dev)
    tok, u, su, st = first.repeat(2), torch.rand(2, device=dev), torch.rand(1, device=dev), starts
    for bad in (dict(tokens=tok.long()), dict(target_probs=p.half()), dict(target_probs=p.t().contiguous().t()),
                dict(draft_probs=p[:, :6]), dict(draft_probs=p.half()), dict(uniforms=su), dict(sample_u=u),
                dict(starts=first[:0]), dict(starts=st.long())):
        a = dict(tokens=tok, target_probs=p, draft_probs=None, uniforms=u, sample_u=su, starts=st)
        a.update(bad)
        with pytest.raises(ValueError):
            paged.verify_drafts(**a)
    cache = paged.PagedCache8(1, hk, d, 2, 2, 64, page_size=16)
    cache.reserve(0, 17)
    with pytest.raises(RuntimeError):
        cache.reserve(1, 1)
    with pytest.raises(RuntimeError):
        cache.reserve(0, 65)
    cache.release(0)
    cache.reserve(1, 32)
