"""Beam search over shared 4-bit pages: every returned continuation rescored as a
sequence of its own (no sharing, no copies), greedy search with one beam, an
exhaustive search where the beams hold every prefix, and the pool's pages back.

Rescoring repeats the same f16 / bf16 roundings on other batch shapes, whose
split sums differ in f32 only; a bf16 rounding that falls the other way moves a
logit by about 2^-8 of its terms, so totals of up to a dozen tokens agree within 0.05.
"""
from __future__ import annotations

import numpy as np
import pytest

from doe_b200 import ops

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from doe_b200.beam import BeamSearch  # noqa: E402
from doe_b200.decoder import Decoder, DecoderConfig  # noqa: E402

CFG = DecoderConfig(hidden=512, heads=4, kv_heads=2, ffn=1024, layers=2, ctx=60, kv_dtype="int4")
PROMPT = [3, 77, 100, 5, 9, 118, 31]


@pytest.mark.parametrize("kv", ["int4", "f16"])
@pytest.mark.parametrize("page", [16, 32])
def test_beams_score_as_sequences_of_their_own(kv, page):
    from dataclasses import replace

    b = BeamSearch(replace(CFG, kv_dtype=kv, page_size=page), 512, 5)
    pages = b.pool.free_pages()
    out = b.search(PROMPT, 12)  # positions 7 to 17: the copied page and, at page 16, a fresh one
    assert b.pool.free_pages() == pages
    assert len(out) == 5 and len({tuple(t) for t, _ in out}) == 5
    scores = [s for _, s in out]
    assert scores == sorted(scores, reverse=True)
    for tokens, s in out:
        assert abs(b.score(PROMPT, tokens) - s) < 0.05
    assert b.pool.free_pages() == pages
    assert [t for t, _ in b.search(PROMPT, 12)] == [t for t, _ in out], "a second search differs"
    b.close()


def test_one_beam_is_greedy():
    b = BeamSearch(CFG, 256, 1)
    (tokens, score), = b.search(PROMPT, 6)
    logits = b._prefill(PROMPT)
    for i, t in enumerate(tokens):
        assert int(logits.argmax()) == t
        if i + 1 < len(tokens):
            logits = b._logits(b.one, [0], [t], len(PROMPT) + i + 1)
    b.pool.release(0)
    assert abs(b.score(PROMPT, tokens) - score) < 0.05
    b.close()


def test_two_steps_match_the_scores_of_every_pair_found():
    """16 beams after two steps: no first token among the 16 best extends better than those kept."""
    b = BeamSearch(CFG, 128, 16)
    out = b.search(PROMPT, 2)
    lp = ops.token_logprobs(b._prefill(PROMPT), top_k=16)
    b.pool.release(0)
    pairs = []
    for t, s in zip(lp.top_ids[0].tolist(), lp.top_logprobs[0].tolist()):
        b._prefill(PROMPT)
        alt = ops.token_logprobs(b._logits(b.one, [0], [t], len(PROMPT) + 1), top_k=16)
        b.pool.release(0)
        pairs += [(s + v, [t, u]) for u, v in zip(alt.top_ids[0].tolist(), alt.top_logprobs[0].tolist())]
    want = sorted(pairs, reverse=True)[:16]
    for (score, _), (_, got) in zip(want, out):
        assert abs(score - got) < 0.02
    b.close()


def test_a_kept_sequence_survives_searches_and_compaction():
    b = BeamSearch(CFG, 256, 3, spare_pages=3)
    keep = 2 * b.beams
    b.pool.reserve(1, 40)  # so that the kept pages are not the first
    for i in range(20):
        b._logits(b.one, [keep], [i + 1], i + 1)
    b._map([keep])
    before = [[x.cpu() for x in ops.paged_read(c, torch.zeros(1, dtype=torch.int32, device="cuda"), 20)] for c in b.caches]
    b.pool.release(1)
    b.search(PROMPT, 8)
    assert b.compact() == 2
    assert b.pool.block_table()[keep].max() == 1
    b._map([keep])
    for c, x in zip(b.caches, before):
        for y, z in zip(ops.paged_read(c, torch.zeros(1, dtype=torch.int32, device="cuda"), 20), x):
            assert torch.equal(y.cpu(), z)
    b.close()


def test_int4_decoder_step_in_a_graph():
    """The decoder makes and reads its own 4-bit caches; a captured step repeats the eager one."""
    cfg = DecoderConfig(hidden=512, heads=4, kv_heads=2, ffn=1024, layers=2, batch=8, ctx=300, kv_dtype="int4")
    d = Decoder(cfg)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x0 = torch.randn((8, 512), generator=g, device="cuda")
    want = d.step(x0.clone()).clone()
    x = x0.clone()
    d.capture(x)
    for _ in range(2):
        x.copy_(x0)
        d.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want)
    d.check()
    f16 = Decoder(DecoderConfig(hidden=512, heads=4, kv_heads=2, ffn=1024, layers=2, batch=8, ctx=300),
                  layers=d.layers)
    # the same weights over f16 caches of the same values
    for c4, c in zip(d.caches, f16.caches):
        k, v = ops.paged_read(c4, torch.zeros(8, dtype=torch.int32, device="cuda"), 300)
        ops.paged_append(c, k, v, torch.zeros(8, dtype=torch.int32, device="cuda"))
    near = f16.step(x0.clone())
    # apart from the new token's own quantisation (one of 301) both attend to the same values
    assert float((near - want).norm() / want.norm()) < 0.01


def test_refusals():
    with pytest.raises(ValueError):
        BeamSearch(CFG, 100, 2)
    with pytest.raises(ValueError):
        BeamSearch(CFG, 128, 17)
    b = BeamSearch(CFG, 128, 2)
    with pytest.raises(ValueError):
        b.search([], 3)
    with pytest.raises(ValueError):
        b.search([1] * 58, 4)
    with pytest.raises(ValueError):
        b.search([1, 128], 4)  # no such token
    with pytest.raises(ValueError):
        b.score([1], [-1])
    assert b.pool.free_pages() == b.pool.num_pages
    b.close()
