"""Beam search on the decoder over a 4-bit paged KV cache.

The operators of serving several continuations of a prompt, as they are used
together:

    Decoder.step                 one token per beam; its attention reads and
                                 appends to 4-bit caches (paged_decode)
    token_logprobs               each beam's alternatives, from the logits
    KvPool.fork / release        the surviving beams share their parents' pages
    KvPool.make_writable,        the last page is copied before beams that
    paged_copy_pages             share it write different tokens into it
    KvPool.compact               pages of finished searches are closed up

    python -m doe_b200.beam --beams 4 --steps 32

The weights are random (there is no checkpoint here); the model is the
decoder block of doe_b200.decoder between an embedding and an output matrix.
"""
from __future__ import annotations

import argparse
from dataclasses import replace

import numpy as np
import torch

from . import ops
from .decoder import Decoder, DecoderConfig
from .kv import KvPool, PagedKVCache


class BeamSearch:
    """A decoder with `beams` sequences whose pages come from one host pool.

    cfg.batch is ignored (beams) and cfg.ctx is the longest sequence.  Every
    layer's cache has the same block table, so one page list serves all."""

    def __init__(self, cfg: DecoderConfig, vocab: int, beams: int, *, seed: int = 4, spare_pages: int = 0, device=None):
        if vocab % 128:
            raise ValueError("vocab must be a multiple of 128 (doe_linear_bf16)")
        if not 1 <= beams <= min(32, ops.abi.LOGPROBS_MAX_TOP // 2):
            raise ValueError("1 to 16 beams: a step takes 2 alternatives per beam")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.cfg, self.vocab, self.beams, self.device = cfg, vocab, beams, dev
        per_seq = -(-cfg.ctx // cfg.page_size)
        # a step holds the old and the new beams' rows at once; their pages are shared but for the last
        self.pool = KvPool(beams * per_seq + beams + spare_pages, cfg.page_size, 2 * beams + 1, per_seq)
        table = self.pool.block_table()[:beams]
        self.caches = [PagedKVCache(num_pages=self.pool.num_pages, page_size=cfg.page_size, num_kv_heads=cfg.kv_heads,
                                    head_dim=cfg.head_dim, block_table=table, kv_dtype=cfg.kv_dtype, device=dev)
                       for _ in range(cfg.layers)]
        self.many = Decoder(replace(cfg, batch=beams), seed=seed, caches=self.caches, device=dev)
        self.one = Decoder(replace(cfg, batch=1), layers=self.many.layers, caches=self.caches, device=dev)
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        self.embed = torch.randn((vocab, cfg.hidden), generator=g, device=dev)
        self.head = (torch.randn((vocab, cfg.hidden), generator=g, device=dev) * cfg.hidden ** -0.5).to(torch.bfloat16)
        self.norm = torch.ones(cfg.hidden, dtype=torch.bfloat16, device=dev)
        self.head_ws = torch.zeros(int(ops.abi.lib().doe_linear_workspace_bytes(vocab, cfg.hidden)), dtype=torch.uint8,
                                   device=dev)

    def _map(self, slots) -> None:
        """The sequences of pool slots `slots` become the caches' rows 0, 1, ..."""
        table = torch.from_numpy(self.pool.block_table()[list(slots)]).to(self.device)
        for c in self.caches:
            c.block_table = table

    def _copy(self, pairs) -> None:
        for c in self.caches:
            ops.paged_copy_pages(c, pairs)

    def _logits(self, dec: Decoder, slots, tokens, length: int) -> torch.Tensor:
        """Appends tokens[i] at position length - 1 of slots[i]: the next tokens' logits, f32."""
        for s in slots:
            self.pool.reserve(s, length)
        self._copy(np.concatenate([self.pool.make_writable(s, length - 1, 1) for s in slots]))
        self._map(slots)
        x = self.embed[torch.as_tensor(tokens, device=self.device)]
        dec.seq_lens.fill_(length)
        dec.step(x)
        out = torch.empty((len(slots), self.vocab), dtype=torch.float32, device=self.device)
        ops.linear(ops.rmsnorm(x, self.norm, self.cfg.eps, status=dec.status), self.head, [out], status=dec.status,
                   ws=self.head_ws)
        return out

    def _prefill(self, prompt) -> torch.Tensor:
        if not prompt or not all(0 <= t < self.vocab for t in prompt):
            raise ValueError("the prompt must be tokens of [0, vocab), one at least")
        for i, t in enumerate(prompt):
            logits = self._logits(self.one, [0], [t], i + 1)
        return logits

    def search(self, prompt: list[int], steps: int) -> list[tuple[list[int], float]]:
        """The `beams` best continuations of `steps` tokens found, best first: (tokens, log probability)."""
        if steps < 1 or len(prompt) + steps - 1 > self.cfg.ctx:
            raise ValueError(f"{len(prompt)} + {steps} tokens do not fit cfg.ctx = {self.cfg.ctx}")
        W = self.beams
        slots, found, scores = [0], [[]], np.zeros(1)
        try:
            logits = self._prefill(prompt)
            for step in range(steps):
                alt = ops.token_logprobs(logits, top_k=min(2 * W, self.vocab))
                total = scores[:, None] + alt.top_logprobs.double().cpu().numpy()
                ids = alt.top_ids.cpu().numpy()
                best = np.argsort(-total, axis=None, kind="stable")[:W]
                parent, col = np.unravel_index(best, total.shape)
                found = [found[p] + [int(ids[p, c])] for p, c in zip(parent, col)]
                scores = total[parent, col]
                if step + 1 == steps:
                    break
                length = len(prompt) + step
                free = [s for s in range(2 * W) if s not in slots][:W]
                for p, s in zip(parent, free):
                    self.pool.fork(slots[p], s, length)
                for s in slots:
                    self.pool.release(s)
                slots = free
                logits = self._logits(self.many, slots, [f[-1] for f in found], length + 1)
        finally:
            for s in range(2 * W):
                self.pool.release(s)
        self.many.check()
        self.one.check()
        return [(f, float(s)) for f, s in zip(found, scores)]

    def score(self, prompt: list[int], tokens: list[int]) -> float:
        """The log probability of `tokens` after `prompt`, decoded as one sequence."""
        if not all(0 <= t < self.vocab for t in tokens) or len(prompt) + len(tokens) - 1 > self.cfg.ctx:
            raise ValueError(f"tokens must be of [0, vocab) and fit cfg.ctx = {self.cfg.ctx} after the prompt")
        given = torch.tensor([[t] for t in tokens], dtype=torch.int32, device=self.device)
        total = torch.zeros(1, dtype=torch.float64, device=self.device)
        try:
            logits = self._prefill(prompt)
            for i in range(len(tokens)):
                total += ops.token_logprobs(logits, given[i]).logprob
                if i + 1 < len(tokens):
                    logits = self._logits(self.one, [0], [tokens[i]], len(prompt) + i + 1)
        finally:
            self.pool.release(0)
        self.one.check()
        return float(total.item())

    def compact(self) -> int:
        """Closes up the live pages (of sequences kept outside a search); the number of pages moved."""
        pairs = self.pool.compact()
        self._copy(pairs)
        return len(pairs)

    def close(self) -> None:
        self.pool.close()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--prompt", type=int, nargs="+", default=[1, 17, 42, 99, 7])
    ap.add_argument("--kv", choices=["f16", "int8", "int4"], default="int4")
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--vocab", type=int, default=32768)
    args = ap.parse_args()
    heads = args.hidden // 128
    cfg = DecoderConfig(hidden=args.hidden, heads=heads, kv_heads=max(1, heads // 4), ffn=4 * args.hidden,
                        layers=args.layers, ctx=len(args.prompt) + args.steps, kv_dtype=args.kv)
    b = BeamSearch(cfg, args.vocab, args.beams)
    for tokens, logprob in b.search(args.prompt, args.steps):
        print(f"{logprob:10.4f}  {' '.join(map(str, tokens))}")
    b.close()


if __name__ == "__main__":
    main()
