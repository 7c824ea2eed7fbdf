"""The serving loop over the paged operators (megakernel_b200.drafted)."""
import numpy as np
import pytest
import torch

from megakernel_b200 import weights as W
from megakernel_b200.drafted import DraftedDecoder, lookup_draft, main
from oracle.qwen3_decode import Qwen3DecodeOracle

from ._common import weights


def test_lookup_draft():
    assert lookup_draft([1, 2, 3, 9, 1, 2, 3], 2) == [9, 1]
    assert lookup_draft([5, 1, 7, 1], 3) == [7, 1]
    assert lookup_draft([4, 8, 4, 9, 4], 1) == [9]            # the latest occurrence
    assert lookup_draft([1, 2, 9, 3, 2, 8, 1, 2], 1) == [9]   # the longer n-gram first
    assert lookup_draft([1, 2, 3], 4) == []
    assert lookup_draft([1], 4) == [] and lookup_draft([1, 1], 0) == []


def rel(a, b):
    return np.linalg.norm(a - b) / np.linalg.norm(b)


@pytest.mark.gpu
@pytest.mark.parametrize("name,kv,tol", [("tiny", "int8", 0.04), ("tiny", "fp8", 0.06), ("qwen3-0.6b-d128", "int8", 0.12)])
def test_forward_against_the_oracle(name, kv, tol):
    """Logits of a prompt fed in uneven pieces, two sequences side by side.

    Tolerance (2-norm, relative): some ten bf16 roundings per layer on the way
    to the logits, each 2^-9 rms at most, add up like sqrt(10 layers) 2^-9: 0.9 %
    for 2 layers, 3.3 % for 28; int8 codes of a page are within half of
    2^-6 of its maximum, about 0.5 % of a value; e4m3 codes within 2^-4, 1.8 %
    rms; averaged by attention these stay below their size.  Twice the sum and
    as much again for the growth of errors through the layers."""
    shape, w, flat, offs = weights(name)
    n = 37
    ids = [W.prompt_ids(shape, n, seed=s) for s in (1, 2)]
    dec = DraftedDecoder(flat, offs, shape, seqs=2, max_seq=64, page_size=16, kv_dtype=kv)
    got = [[], []]
    for cut in ((0, 0, 20, 1), (20, 1, 21, 30), (21, 30, 37, 37)):
        a, b, a2, b2 = cut
        logits, starts = dec.forward([ids[0][a:a2], ids[1][b:b2]], [a, b])
        got[0].append(logits[:a2 - a].cpu().numpy())
        got[1].append(logits[a2 - a:].cpu().numpy())
    for b in range(2):
        o = Qwen3DecodeOracle(shape, w, kv_bf16=False, max_seq=64, device="cuda")
        _, want, _ = o.run(ids[b], n)
        assert rel(np.concatenate(got[b]), want) < tol


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["fp8", "int8"])
def test_generate_greedy_with_and_without_drafts(kv):
    """Every generated token is the most likely one, or within the logits' noise
    of it, whether it was drafted or not; drafts take fewer steps.  The noise is
    the tolerance above of the logits' spread, on both logits, four deviations
    each."""
    shape, w, flat, offs = weights("tiny")
    dec = DraftedDecoder(flat, offs, shape, seqs=3, max_seq=128, page_size=16, kv_dtype=kv)
    base = W.prompt_ids(shape, 9, seed=3)
    prompts = [base * 3, W.prompt_ids(shape, 5, seed=4), base]
    steps = {}
    for drafts in (0, 4):
        out, steps[drafts] = dec.generate(prompts, 60, max_drafts=drafts)
        assert [len(t) for t in out] == [60] * 3
        for p, t in zip(prompts, out):
            logits = dec.forward([p + t, [], []], [0, 0, 0])[0][len(p) - 1:-1]
            noise = 0.06 * logits.std(1, correction=0)
            picked = logits.gather(1, torch.tensor(t, device=logits.device)[:, None])[:, 0]
            assert (logits.amax(1) - picked <= 8 * noise).all()
    assert steps[0] == 60 and steps[4] < 60


@pytest.mark.gpu
def test_generate_samples_and_repeats():
    shape, w, flat, offs = weights("tiny")
    dec = DraftedDecoder(flat, offs, shape, seqs=2, max_seq=64, page_size=32)
    prompts = [W.prompt_ids(shape, 7, seed=5) * 2, W.prompt_ids(shape, 3, seed=6)]
    a, _ = dec.generate(prompts, 20, temperature=1.0, seed=11)
    b, _ = dec.generate(prompts, 20, temperature=1.0, seed=11)
    c, _ = dec.generate(prompts, 20, temperature=1.0, seed=12)
    assert a == b and a != c
    assert all(0 <= t < shape.vocab for s in a for t in s)
    with pytest.raises(ValueError):
        dec.generate(prompts, 60)
    with pytest.raises(ValueError):
        dec.generate([[]], 2)


@pytest.mark.gpu
def test_command():
    assert main(["--tokens", "8", "--seqs", "2", "--prompt", "6"]) == 0
