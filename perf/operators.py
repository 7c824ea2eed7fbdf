"""Measured cases of the paged 8-bit serving operators, with their plain forms.

The operators are the parts of one serving step with drafted tokens: the norm
and rotation of queries and keys, the write of keys and values into a paged
8-bit cache and its read-back, attention over that cache, and the verification
of drafted tokens.  `run` computes them in elementary torch operations, or,
where `own` is true, through megakernel_b200.paged.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
QMAX = {"fp8": 448.0, "int8": 127.0}
FIX = 36    # probabilities are held in units of 2^-36
FIXU = 24   # random numbers in units of 2^-24


# ---- cases --------------------------------------------------------------------
# Head counts (16 query heads over 8 key/value heads), head sizes 64 and 128, the
# vocabulary of 151,936, 64 sequences of about 1,024 to 1,280 tokens, one sequence
# at position 639 and contexts of 8,192 are this repository's shapes and workloads.

def listed():
    return [
        # one token of one sequence: the launch is all that counts
        dict(name="norm_rope_one", op="norm_rope", rows=1, hq=16, hk=8, d=64, type="bf16", packed=True),
        # 64 prompts of about 1,024 tokens at once, sliced out of a packed projection
        dict(name="norm_rope_prompts", op="norm_rope", rows=65531, hq=16, hk=8, d=64, type="bf16", packed=True),
        # one new token for each of 64 sequences, into pages that hold earlier tokens
        dict(name="append_step", op="append", seqs=64, rows_lo=1, rows_hi=1, first_lo=1024, first_hi=1279,
             hk=8, d=64, page=64, fmt="fp8", type="bf16"),
        # 64 prompts of unequal length written at once
        dict(name="append_prompts", op="append", seqs=64, rows_lo=897, rows_hi=1151, first_lo=0, first_hi=37,
             hk=8, d=128, page=32, fmt="int8", type="bf16"),
        # the 640 positions of one sequence back in 16 bits
        dict(name="read_one", op="read", seqs=1, rows_lo=640, rows_hi=640, first_lo=0, first_hi=0,
             hk=8, d=64, page=64, fmt="fp8", type="bf16"),
        # sixteen long contexts, each from an odd position on
        dict(name="read_long", op="read", seqs=16, rows_lo=7001, rows_hi=8191, first_lo=1, first_hi=61,
             hk=8, d=128, page=16, fmt="int8", type="f16"),
        # one token of one sequence at position 639: latency
        dict(name="attend_one", op="attend", seqs=1, rows_lo=1, rows_hi=1, len_lo=640, len_hi=640, hq=16, hk=8, d=64,
             page=64, fmt="fp8", type="bf16", window=0, lse=False),
        # a decode step of 64 sequences of 1,024 to 1,280 positions
        dict(name="attend_step", op="attend", seqs=64, rows_lo=1, rows_hi=1, len_lo=1024, len_hi=1280, hq=16, hk=8,
             d=64, page=64, fmt="fp8", type="bf16", window=0, lse=False),
        # the verifying step of 24 long contexts: the last token and 2 to 7 drafted ones each
        dict(name="attend_drafts", op="attend", seqs=24, rows_lo=3, rows_hi=8, len_lo=4099, len_hi=8192, hq=16, hk=8,
             d=128, page=16, fmt="int8", type="f16", window=0, lse=True),
        # a chunk of a prompt after its earlier chunks, for four sequences
        dict(name="attend_prompt", op="attend", seqs=4, rows_lo=1900, rows_hi=2048, len_lo=2048, len_hi=8192, hq=16,
             hk=8, d=128, page=64, fmt="fp8", type="bf16", window=0, lse=False),
        # one sequence, four drafted tokens out of a lookup (no draft distribution), a small vocabulary
        dict(name="verify_one", op="verify", seqs=1, rows_lo=5, rows_hi=5, vocab=2048, draft_probs=False, near=0.5),
        # 64 sequences with up to seven drafts of a draft model
        dict(name="verify_step", op="verify", seqs=64, rows_lo=3, rows_hi=8, vocab=151936, draft_probs=True, near=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "read", "attend", "attend", "verify"])
    d, page = rng.choice([64, 128]), rng.choice([16, 32, 64])
    hk = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 2, 4, 8])
    fmt, kind = rng.choice(["fp8", "int8"]), rng.choice(["bf16", "f16"])
    if op == "norm_rope":
        return dict(op=op, rows=_log(rng, 1, 32768), hq=hk * group if hk * group <= 24 else 24, hk=hk, d=d,
                    type=rng.choice(["bf16", "f16", "f32"]), packed=rng.random() < 0.5)
    if op in ("append", "read"):
        seqs = _log(rng, 1, 64)
        most = max(1, min(8192, 60000 // seqs))
        lo = _log(rng, 1, most)
        hi = min(most, lo + rng.randrange(0, 1 + lo // 4))
        first = rng.choice([0, rng.randrange(0, 300)])
        return dict(op=op, seqs=seqs, rows_lo=lo, rows_hi=hi, first_lo=first, first_hi=first + rng.randrange(0, 70),
                    hk=hk, d=d, page=page, fmt=fmt, type=rng.choice(["bf16", "f16", "f32"]))
    if op == "attend":
        form = rng.choice(["step", "drafts", "prompt"])
        lse, window = rng.random() < 0.5, rng.choice([0, 0, 0, rng.randrange(1, 2000)])
        if form == "prompt":
            seqs, rows = rng.choice([1, 2, 3]), _log(rng, 17, 2000)
            length = rows + _log(rng, 1, 5000)
        else:
            seqs, rows = _log(rng, 1, 64), 1 if form == "step" else rng.randrange(2, 17)
            length = rows + _log(rng, 1, max(2, 160000 // seqs if seqs > 5 else 32000))
        return dict(op=op, seqs=seqs, rows_lo=max(1, rows - rng.randrange(0, 3)), rows_hi=rows,
                    len_lo=max(rows, length // 2), len_hi=length, hq=hk * group, hk=hk, d=d, page=page, fmt=fmt,
                    type=kind, window=window, lse=lse)
    seqs, rows = _log(rng, 1, 64), rng.randrange(1, 9)
    return dict(op=op, seqs=seqs, rows_lo=max(1, rows - rng.randrange(0, 4)), rows_hi=rows,
                vocab=_log(rng, 500, 151936), draft_probs=rng.random() < 0.7, near=rng.choice([0.2, 0.5, 1.5]))


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, out of order."""
    return [lo + (hi - lo) * ((b * 7919) % n) // max(n - 1, 1) for b in range(n)]


def _rows(case):
    return _spread(case["rows_lo"], case["rows_hi"], case["seqs"])


def _seen(case, rows, lens):
    """Query-key pairs of one head that the causal mask and the window leave."""
    n = 0
    for r, length in zip(rows, lens):
        p = np.arange(length - r, length) + 1
        n += int(np.minimum(p, case["window"]).sum() if case["window"] else p.sum())
    return n


def work(case):
    op = case["op"]
    if op == "norm_rope":
        n = case["rows"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * n * SIZE[case["type"]] + case["rows"] * (4 * case["d"] + 4), "flops": 10 * n}
    rows = _rows(case)
    if op == "append":  # the new rows in 16 or 32 bits in, their codes out, then the pages' values read back
        first = _spread(case["first_lo"], case["first_hi"], case["seqs"])
        n = sum(rows) * 2 * case["hk"] * case["d"]
        back = sum(r + f % case["page"] for r, f in zip(rows, first)) * 2 * case["hk"] * case["d"]
        return {"bytes": n * (SIZE[case["type"]] + 1) + back * (1 + SIZE[case["type"]]), "flops": 4 * n + back}
    if op == "read":
        n = sum(rows) * 2 * case["hk"] * case["d"]
        return {"bytes": n * (1 + SIZE[case["type"]]), "flops": n}
    if op == "attend":
        lens = _spread(case["len_lo"], case["len_hi"], case["seqs"])
        held = sum(min(n, case["window"] + r - 1) if case["window"] else n for r, n in zip(rows, lens))
        io = sum(rows) * case["hq"] * case["d"] * 4
        return {"bytes": held * 2 * case["hk"] * case["d"] + io,
                "flops": 4 * case["d"] * case["hq"] * _seen(case, rows, lens)}
    # one target row, and one draft row where a draft is refused (taken as always)
    n = case["seqs"] * case["vocab"]
    return {"bytes": n * 4 * (2 if case["draft_probs"] and case["rows_hi"] > 1 else 1), "flops": 4 * n}


# ---- inputs ---------------------------------------------------------------------

def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(rows):
    return _ints([0] + list(np.cumsum(rows)))


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _kv(gen, rows, hk, d):
    """Keys with a few strong channels, values whose size differs by token."""
    k = _normal(gen, rows, hk, d) * (1 + 3 * (torch.rand(hk, d, generator=gen, device=DEV) < 0.05))
    v = _normal(gen, rows, hk, d) * torch.exp(0.5 * _normal(gen, rows, 1, 1))
    return k, v


def _pool(case, gen, lens, room=0):
    """A pool of pages in random order that holds lens[b] tokens of each sequence and has room for
    `room`; what no token wrote yet holds leftovers: NaN (fp8) or the lowest code (int8)."""
    hk, d, page, fmt = case["hk"], case["d"], case["page"], case["fmt"]
    most = max(1, -(-max(max(lens), room) // page))
    total = len(lens) * most
    order = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
    codes = torch.empty(total, 2, hk, page, d, dtype=torch.int8, device=DEV)
    scales = torch.empty(total, 2, hk, device=DEV)
    held = _ints(lens)
    stale = torch.tensor(0x7F if fmt == "fp8" else -128, dtype=torch.int8, device=DEV)
    for j in range(0, total, 1024):  # some pages at a time
        at = torch.arange(j, min(j + 1024, total), device=DEV)
        k, v = _kv(gen, at.numel() * page, hk, d)
        x = torch.stack([k, v], 1).view(at.numel(), page, 2, hk, d).permute(0, 2, 3, 1, 4)
        there = (at % most)[:, None] * page + torch.arange(page, device=DEV) < held[at // most][:, None]
        x = torch.where(there[:, None, None, :, None], x, 0.0)
        scale = _scale_of(x.abs().amax((3, 4)), fmt)
        code = _codes_of(x / scale[..., None, None], fmt).view(torch.int8)
        codes[order[at].long()] = torch.where(there[:, None, None, :, None], code, stale)
        scales[order[at].long()] = torch.where(there.any(1)[:, None, None], scale, 2.0 ** 20)
    return codes.view(torch.float8_e4m3fn) if fmt == "fp8" else codes, scales, order.view(-1, most)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) * 1000003 + 17)
    st = dict(case=dict(case))
    op = case["op"]
    if op == "norm_rope":
        t, hq, hk, d, kind = case["rows"], case["hq"], case["hk"], case["d"], TYPES[case["type"]]
        if case["packed"]:  # q, k and v of a token side by side, as one projection leaves them
            x = (2 * _normal(gen, t, (hq + 2 * hk) * d)).to(kind)
            st["q"] = x[:, :hq * d].unflatten(1, (hq, d))
            st["k"] = x[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
        else:
            st["q"], st["k"] = (2 * _normal(gen, t, hq, d)).to(kind), (2 * _normal(gen, t, hk, d)).to(kind)
        st["q_gain"], st["k_gain"] = ((1 + 0.2 * _normal(gen, d)).to(kind) for _ in range(2))
        angle = torch.arange(8448, device=DEV)[:, None] * 1.0e6 ** (-torch.arange(0, d, 2, device=DEV) / d)
        st["cos"], st["sin"] = angle.cos(), angle.sin()
        st["positions"] = torch.randint(0, 8448, (t,), generator=gen, device=DEV, dtype=torch.int32)
        return st
    rows = _rows(case)
    st["starts"], total = _starts(rows), sum(rows)
    if op in ("append", "read"):
        first = _spread(case["first_lo"], case["first_hi"], case["seqs"])
        lens = [f + r for f, r in zip(first, rows)]
        page = case["page"]
        held = first if op == "append" else lens
        st["codes"], st["scales"], st["table"] = _pool(case, gen, held, max(lens))
        if op == "append":
            k, v = _kv(gen, total, case["hk"], case["d"])
            st["k"], st["v"] = k.to(TYPES[case["type"]]), v.to(TYPES[case["type"]])
            # the read-back begins with the page that the first new token falls into
            back = [f // page * page for f in first]
            st["back_first"] = _ints(back)
            st["back_starts"] = _starts([n - f for n, f in zip(lens, back)])
            st["back_rows"] = sum(lens) - sum(back)
            st["windows"] = max(-(-(f % page + r) // page) for f, r in zip(first, rows))
        st["first"], st["rows"], st["longest"] = _ints(first), total, max(rows)
        return st
    if op == "attend":
        lens = _spread(case["len_lo"], case["len_hi"], case["seqs"])
        st["codes"], st["scales"], st["table"] = _pool(case, gen, lens)
        st["first"] = _ints([n - r for n, r in zip(lens, rows)])
        st["q"] = (1.5 * _normal(gen, total, case["hq"], case["d"])).to(TYPES[case["type"]])
        st["longest"] = max(rows)
        return st
    v = case["vocab"]
    logits = 2.5 * _normal(gen, total, v)
    st["target"] = torch.softmax(logits, 1)
    draft = torch.softmax(logits + case["near"] * _normal(gen, total, v), 1)
    del logits
    picked = torch.multinomial(draft, 1, generator=gen)[:, 0].to(torch.int32)
    # row i of a sequence scores the token after it: draft i + 1 was picked from row i
    st["tokens"] = torch.roll(picked, 1)
    st["draft"] = draft if case["draft_probs"] else None
    st["uniforms"] = torch.rand(total, generator=gen, device=DEV)
    st["sample_u"] = torch.rand(case["seqs"], generator=gen, device=DEV)
    st["longest"] = max(rows)
    return st


# ---- plain forms -------------------------------------------------------------------

def _pow2(e):
    """2^e for whole e from -126 to 127."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _scale_of(amax, fmt):
    """The smallest power of two (at least 2^-126) that brings amax into the format's range."""
    m, e = torch.frexp(amax.float())
    e = e - 9 + (m > 0.875).int() if fmt == "fp8" else e - 7 + (m > 0.9921875).int()
    e = torch.where(amax > 0, e, -126).clamp(min=-126)
    return _pow2(e)


def _codes_of(x, fmt):
    """x (in units of the scale) to the nearest code, ties to even."""
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8)
    _, e = torch.frexp(x)
    step = _pow2(e.clamp(min=-5) - 4)  # 3 bits after the leading one; 2^-9 at least
    return (torch.round(x / step) * step).clamp(-448, 448).to(torch.float8_e4m3fn)


def _values(codes, scales, pages):
    """The values that the codes of some pages stand for: [..., 2, heads, page, d] in 32 bits."""
    c = codes.view(torch.int8)[pages.long()].view(codes.dtype).float()
    return c * scales[pages.long()][..., None, None]


def _places(st):
    """Sequence and position of each packed row."""
    t = torch.arange(st["rows"] if "rows" in st else st["q"].shape[0], device=DEV, dtype=torch.int32)
    seq = torch.searchsorted(st["starts"][1:].contiguous(), t, right=True)
    return seq, st["first"][seq] + t - st["starts"][seq]


def _plain_norm_rope(st):
    def one(x, gain):
        x = x.float()
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gain.float()
        c, s = (st[n][st["positions"].long()][:, None] for n in ("cos", "sin"))
        a, b = y.chunk(2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    return one(st["q"], st["q_gain"]).to(st["q"].dtype), one(st["k"], st["k_gain"]).to(st["k"].dtype)


def _plain_append(st):
    case, page = st["case"], st["case"]["page"]
    b = st["first"].shape[0]
    count = st["starts"][1:] - st["starts"][:-1]
    w = torch.arange(st["windows"], device=DEV)
    base = st["first"].div(page, rounding_mode="floor")
    # position of each slot of the pages that a sequence's new tokens touch
    pos = ((base[:, None] + w)[:, :, None] * page + torch.arange(page, device=DEV))
    new = (pos >= st["first"][:, None, None]) & (pos < (st["first"] + count)[:, None, None])
    old = (pos < st["first"][:, None, None])
    touched = new.any(2)
    pages = st["table"][torch.arange(b, device=DEV)[:, None], (base[:, None] + w).clamp(max=st["table"].shape[1] - 1).long()]
    row = (st["starts"][:-1, None, None] + pos - st["first"][:, None, None]).clamp(0, st["rows"] - 1).long()
    x = torch.stack([st["k"], st["v"]], 1).float()[row]               # [b, w, page, 2, hk, d]
    x = torch.where(new[..., None, None, None], x, 0.0).permute(0, 1, 3, 4, 2, 5)
    need = _scale_of(x.abs().amax((4, 5)), case["fmt"])
    was = st["scales"][pages.long()]
    scale = torch.where(old.any(2)[..., None, None], torch.maximum(need, was), need)
    held = _values(st["codes"], st["scales"], pages)
    mask_new, mask_old = (m[:, :, None, None, :, None] for m in (new, old))
    full = torch.where(mask_new, x, torch.where(mask_old, held, 0.0))
    codes = _codes_of(full / scale[..., None, None], case["fmt"]).view(torch.int8)
    codes = torch.where(mask_new | mask_old, codes, st["codes"].view(torch.int8)[pages.long()])
    at = pages[touched].long()
    st["codes"].view(torch.int8)[at] = codes[touched]
    st["scales"][at] = scale[touched]


def _plain_read(st):
    seq, pos = _places(st)
    page = st["case"]["page"]
    at = st["table"][seq, pos.div(page, rounding_mode="floor").long()].long()
    slot = (pos % page).long()
    c = st["codes"].view(torch.int8)[at, :, :, slot].view(st["codes"].dtype).float()   # [t, 2, hk, d]
    x = (c * st["scales"][at][..., None]).to(TYPES[st["case"]["type"]])
    return x[:, 0].contiguous(), x[:, 1].contiguous()


def _plain_attend(st):
    case = st["case"]
    b, d, hk, group = st["first"].shape[0], case["d"], case["hk"], case["hq"] // case["hk"]
    count = st["starts"][1:] - st["starts"][:-1]
    i = torch.arange(st["longest"], device=DEV)
    row = (st["starts"][:-1, None] + i).clamp(max=st["q"].shape[0] - 1).long()
    q = st["q"].float()[row].view(b, st["longest"], hk, group, d).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
    kv = _values(st["codes"], st["scales"], st["table"])              # [b, pages, 2, hk, page, d]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, b, hk, -1, d)
    j = torch.arange(kv.shape[3], device=DEV)
    held = j < (st["first"] + count)[:, None]
    kv = torch.where(held[None, :, None, :, None], kv, 0.0)
    pos = st["first"][:, None] + i
    seen = (j <= pos[..., None]) & held[:, None]
    if case["window"]:
        seen = seen & (j > pos[..., None] - case["window"])
    s = torch.matmul(q, kv[0].transpose(2, 3)) * d ** -0.5
    s = s.view(b, hk, st["longest"], group, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    s = s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    out = torch.matmul(s.flatten(2, 3), kv[1]).view(b, hk, st["longest"], group, d)
    out = torch.where(total > 0, out / total, 0.0)
    keep = i < count[:, None]
    out = out.permute(0, 2, 1, 3, 4).reshape(b, st["longest"], hk * group, d)[keep].to(st["q"].dtype)
    if not case["lse"]:
        return out
    lse = (top + torch.log(total))[..., 0].permute(0, 2, 1, 3).reshape(b, st["longest"], hk * group)[keep]
    return out, lse


def _fixed(p):
    return torch.round(torch.where(p > 0, p.clamp(max=1.0), 0.0) * 2.0 ** FIX).to(torch.int64)


def _fixed_u(u):
    return torch.floor(u * 2.0 ** FIXU).to(torch.int64)


def _plain_verify(st):
    starts = st["starts"].long()
    count, most = starts[1:] - starts[:-1], st["longest"]
    b, total = count.shape[0], st["tokens"].shape[0]
    i = torch.arange(most, device=DEV)
    row = (starts[:-1, None] + i).clamp(max=total - 1)
    token = st["tokens"].long()[(row + 1).clamp(max=total - 1)]       # the draft that row i scores
    p = _fixed(st["target"][row, token])
    q = _fixed(st["draft"][row, token]) if st["draft"] is not None else torch.full_like(p, 1 << FIX)
    ok = (_fixed_u(st["uniforms"])[row] * q < (p << FIXU)) & (i < count[:, None] - 1)
    accepted = ok.long().cumprod(1).sum(1)
    r = (starts[:-1] + accepted).clamp(max=total - 1)
    weight = _fixed(st["target"][r])
    refused = (accepted < count - 1)[:, None]
    taken = token.gather(1, accepted[:, None])
    if st["draft"] is not None:
        less = _fixed(st["draft"][r])
    else:
        less = torch.zeros_like(weight).scatter_(1, taken, 1 << FIX)
    rest = torch.where(refused, (weight - less).clamp(min=0), weight)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, weight)
    upto = rest.cumsum(1)
    bar = (_fixed_u(st["sample_u"]) * upto[:, -1]) >> FIXU
    sampled = (upto <= bar[:, None]).sum(1)
    sampled = torch.where(upto[:, -1] > 0, sampled, -1)
    out = torch.where(i < accepted[:, None], token, torch.where(i == accepted[:, None], sampled[:, None], -1))
    return out[i < count[:, None]].to(torch.int32), accepted.to(torch.int32)


def run(st):
    op = st["case"]["op"]
    if own:
        return _run_own(st, op)
    if op == "norm_rope":
        return _plain_norm_rope(st)
    if op == "append":
        _plain_append(st)
        back = dict(st, starts=st["back_starts"], first=st["back_first"], rows=st["back_rows"])
        return _plain_read(back) + (st["scales"],)
    if op == "read":
        return _plain_read(st)
    if op == "attend":
        return _plain_attend(st)
    return _plain_verify(st)


def _run_own(st, op):
    from megakernel_b200 import paged
    case = st["case"]
    if op == "norm_rope":
        return paged.qk_norm_rope(st["q"], st["k"], st["q_gain"], st["k_gain"], st["cos"], st["sin"],
                                  st["positions"], eps=1e-6)
    if op == "append":
        paged.kv8_append(st["codes"], st["scales"], st["k"], st["v"], st["table"], st["starts"], st["first"])
        return paged.kv8_read(st["codes"], st["scales"], st["table"], st["back_starts"], st["back_first"],
                              st["back_rows"], dtype=TYPES[case["type"]]) + (st["scales"],)
    if op == "read":
        return paged.kv8_read(st["codes"], st["scales"], st["table"], st["starts"], st["first"], st["rows"],
                              dtype=TYPES[case["type"]])
    if op == "attend":
        return paged.kv8_attend(st["q"], st["codes"], st["scales"], st["table"], st["starts"], st["first"],
                                window=case["window"], return_lse=case["lse"])
    return paged.verify_drafts(st["tokens"], st["target"], st["draft"], st["uniforms"], st["sample_u"], st["starts"])


# ---- 64-bit definitions ----------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"norm_rope": _exact_norm_rope, "append": _exact_append, "read": _exact_read, "attend": _exact_attend,
            "verify": _exact_verify}[case["op"]](case, st)


def _exact_norm_rope(case, st):
    got = []
    half = case["d"] // 2
    at = st["positions"].cpu().long()
    cos, sin = st["cos"].cpu().double()[at].to(DEV), st["sin"].cpu().double()[at].to(DEV)
    for x, gain in ((st["q"], st["q_gain"]), (st["k"], st["k_gain"])):
        x = x.double()
        norm = torch.sqrt(torch.linalg.vector_norm(x, dim=2, keepdim=True) ** 2 / case["d"] + 1e-6)
        y = gain.double() * (x / norm)
        o = torch.empty_like(y)
        o[..., :half] = y[..., :half] * cos.unsqueeze(1) - y[..., half:] * sin.unsqueeze(1)
        o[..., half:] = y[..., half:] * cos.unsqueeze(1) + y[..., :half] * sin.unsqueeze(1)
        got.append(o)
    return tuple(got)


def _dequantised(st, b, upto):
    """Keys and values of the first `upto` positions of sequence b, in 64 bits: [upto, 2, heads, d]."""
    page = st["case"]["page"]
    n = -(-upto // page)
    ids = st["table"][b, :n].long()
    c = st["codes"].view(torch.int8)[ids].view(st["codes"].dtype).double()
    x = c * st["scales"].double()[ids][:, :, :, None, None]
    return x.permute(0, 3, 1, 2, 4).reshape(n * page, *x.shape[1:3], x.shape[4])[:upto]


def _nearest_code(x, fmt):
    if fmt == "int8":
        return torch.round(x)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    e = e + ((x.abs() >= torch.exp2(e + 1)).double()) - (x.abs().clamp(min=2.0 ** -6) < torch.exp2(e)).double()
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_append(case, st):
    page, fmt = case["page"], case["fmt"]
    scales = st["scales"].double().clone()
    starts, first = st["starts"].tolist(), st["first"].tolist()
    table = st["table"].tolist()
    new = torch.stack([st["k"], st["v"]], 1).double()
    parts = []
    for b in range(case["seqs"]):
        f, n = first[b], starts[b + 1] - starts[b]
        begin = f // page * page
        held = _dequantised(st, b, f)[begin:] if f > begin else new[:0]
        x = torch.cat([held, new[starts[b]:starts[b + 1]]])
        pages = -(-x.shape[0] // page)
        pad = torch.zeros(pages * page, *x.shape[1:], dtype=torch.float64, device=DEV)
        pad[:x.shape[0]] = x
        fresh = pad.clone()
        fresh[:f - begin] = 0  # what was held keeps its page's scale, or grows with it
        tops = fresh.view(pages, page, *x.shape[1:]).abs().amax((1, 4))       # [pages, 2, heads]
        e = torch.ceil(torch.log2(tops.clamp(min=2.0 ** -140) / QMAX[fmt]))
        e = torch.where(tops > QMAX[fmt] * torch.exp2(e), e + 1, e)
        e = torch.where(tops <= QMAX[fmt] * torch.exp2(e - 1), e - 1, e).clamp(min=-126)
        sc = torch.exp2(e)
        ids = torch.tensor(table[b][begin // page:begin // page + pages], device=DEV)
        if f > begin:
            sc[0] = torch.maximum(sc[0], scales[ids[0]])
        scales[ids] = sc
        unit = sc.repeat_interleave(page, 0)[..., None]
        parts.append((_nearest_code(pad / unit, fmt) * unit)[:x.shape[0]])
    out = torch.cat(parts)
    return out[:, 0], out[:, 1], scales


def _exact_read(case, st):
    starts, first = st["starts"].tolist(), st["first"].tolist()
    x = torch.cat([_dequantised(st, b, first[b] + starts[b + 1] - starts[b])[first[b]:] for b in range(case["seqs"])])
    return x[:, 0], x[:, 1]


def _exact_attend(case, st):
    group = case["hq"] // case["hk"]
    starts, first = st["starts"].tolist(), st["first"].tolist()
    outs, lses = [], []
    for b in range(case["seqs"]):
        n = starts[b + 1] - starts[b]
        kv = _dequantised(st, b, first[b] + n)
        p = torch.arange(first[b], first[b] + n, device=DEV)[:, None]
        j = torch.arange(first[b] + n, device=DEV)[None]
        hidden = j > p
        if case["window"]:
            hidden = hidden | (p - j >= case["window"])
        heads, ls = [], []
        for h in range(case["hq"]):
            s = st["q"][starts[b]:starts[b + 1], h].double() @ kv[:, 0, h // group].T / math.sqrt(case["d"])
            s[hidden] = -math.inf
            ls.append(torch.logsumexp(s, 1))
            heads.append(torch.exp(s - ls[-1][:, None]) @ kv[:, 1, h // group])
        outs.append(torch.stack(heads, 1))
        lses.append(torch.stack(ls, 1))
    return (torch.cat(outs), torch.cat(lses)) if case["lse"] else torch.cat(outs)


def _exact_verify(case, st):
    starts, tokens = st["starts"].tolist(), st["tokens"].tolist()
    u, su = st["uniforms"].double().cpu().numpy(), st["sample_u"].double().cpu().numpy()
    got, taken = [], []

    def whole(row):
        x = row.double().cpu().numpy()
        return np.rint(np.clip(x, 0.0, 1.0) * 2.0 ** FIX).astype(np.int64)

    for b in range(case["seqs"]):
        lo, n = starts[b], starts[b + 1] - starts[b]
        out, a = [], 0
        while True:
            p = whole(st["target"][lo + a])
            if a == n - 1:
                rest = p
                break
            x = tokens[lo + a + 1]
            if st["draft"] is not None:
                q = whole(st["draft"][lo + a])
            else:
                q = np.zeros_like(p)
                q[x] = 1 << FIX
            if int(u[lo + a] * 2.0 ** FIXU) * int(q[x]) < int(p[x]) << FIXU:
                out.append(x)
                a += 1
                continue
            rest = np.maximum(p - q, 0)
            if rest.sum() == 0:
                rest = p
            break
        upto = np.cumsum(rest)
        bar = (int(su[b] * 2.0 ** FIXU) * int(upto[-1])) >> FIXU
        out.append(int(np.searchsorted(upto, bar, side="right")) if upto[-1] > 0 else -1)
        got += out + [-1] * (n - len(out))
        taken.append(a)
    return (torch.tensor(got, dtype=torch.int32), torch.tensor(taken, dtype=torch.int32))
