"""Speculative decoding rounds on a paged cache with one tiny layer of random weights.

What a serving loop calls in one round, in order:

* ``pages_extend``: room for the round's rows in the lanes' caches;
* ``norm_rotate_append``: the rows' queries, and their keys and values put there;
* ``prefix_attention``: the rows (a verification tree each) over the lanes' caches,
  whose system prompt all lanes share;
* ``process_logits``: the lanes' penalties, each row's drafted ancestors in its
  history, a grammar's masks;
* ``greedy_packet``: every row's token, and from these each lane's accepted path;
* ``keep_rows``, ``pages_truncate``: the cache cut back to that path.

    python examples/speculative_round.py [--lanes 4] [--rounds 6]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np
import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import voidinfer_amd as vi

HEADS, KV_HEADS, DIM, PAGE, VOCAB, WIDTH = 8, 2, 64, 16, 1009, 256
ALLOWED_EVERY = 3   # the toy grammar: after token t, tokens congruent to t modulo 3 may not follow


class Layer:
    """Random weights of one layer, and the rotation's angles."""

    def __init__(self, seed: int, device):
        g = torch.Generator(device="cpu").manual_seed(seed)
        rand = lambda *s: (torch.randn(*s, generator=g) / s[-1] ** 0.5).to(torch.bfloat16).to(device)  # noqa: E731
        self.embed = (rand(VOCAB, WIDTH) * WIDTH ** 0.5).contiguous()
        # the one layer reads embeddings: every token's projection, from one product (a library product's rounding
        # may depend on how many rows it has)
        self.w = rand((HEADS + 2 * KV_HEADS) * DIM, WIDTH)
        self.qkv = self.embed @ self.w.T
        self.out, self.head = rand(WIDTH, HEADS * DIM), rand(VOCAB, WIDTH)
        self.q_weight = self.k_weight = torch.ones(DIM, dtype=torch.bfloat16, device=device)
        angle = torch.arange(4096)[:, None] * 10000.0 ** (-torch.arange(0, DIM, 2) / DIM)
        self.cos, self.sin = angle.cos().float().to(device), angle.sin().float().to(device)


class Lanes:
    """Lanes that share a system prompt: their caches, histories and grammar."""

    def __init__(self, layer: Layer, lanes: int, prompt: list[int], device, pages: int = 256):
        self.layer, self.device, self.n = layer, device, lanes
        i32 = lambda *s, fill=0: torch.full(s, fill, dtype=torch.int32, device=device)  # noqa: E731
        self.pool = torch.zeros(1, 2, pages, KV_HEADS, PAGE, DIM, dtype=torch.bfloat16, device=device)
        self.refs, self.status = i32(pages), i32(3)
        self.tables, self.lengths = i32(lanes, 4096 // PAGE, fill=-1), i32(lanes)
        self.state = vi.PenaltyState(lanes, VOCAB, 4096, device=device)
        self.params = vi.params_array(lanes, repetition_penalty=1.1, presence_penalty=0.2)
        self.masks = self._grammar()
        self.ids = torch.arange(lanes, dtype=torch.int32, device=device)
        # the prompt once, in lane 0; the others fork it
        self.shared = len(prompt)
        self.rows([prompt], [len(prompt) * [0]], only=1)
        if lanes > 1:
            vi.pages_fork(self.refs, self.tables, self.lengths, i32(lanes - 1), self.ids[1:].contiguous(), PAGE, self.status)

    def _grammar(self) -> torch.Tensor:
        words = -(-VOCAB // 32)
        bits = np.zeros((ALLOWED_EVERY, words * 32), dtype=np.uint8)
        for r in range(ALLOWED_EVERY):
            bits[r, :VOCAB] = np.arange(VOCAB) % ALLOWED_EVERY != r
        return torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32).copy()).to(self.device)

    def rows(self, tokens: list[list[int]], parents: list[list[int]], only: int | None = None) -> np.ndarray:
        """One step: per lane its rows' tokens and each row's parent row (its own index for the first; a prompt's
        rows follow one another).  Returns the rows' greedy tokens; the cache holds every row."""
        n = self.n if only is None else only
        dev, layer = self.device, self.layer
        i32 = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=dev)  # noqa: E731
        counts = [len(t) for t in tokens]
        offsets, flat = np.concatenate([[0], np.cumsum(counts)]), i32([x for t in tokens for x in t])
        context = self.lengths[:n].clone()
        ids = self.ids[:n]
        vi.pages_extend(self.refs, self.tables, self.lengths, ids, context + i32(counts), self.pool, self.status)
        x = layer.embed[flat.long()]
        q, k, v = (y.view(len(flat), -1, DIM) for y in layer.qkv[flat.long()].split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], 1))
        chain = max(counts) > 64            # a prompt: plain causal rows
        seen, depth = [], []
        for p in parents:
            bits, d = [], []
            for j, up in enumerate(p):
                bits.append(1 << j if j == 0 else (bits[up] | 1 << j) if not chain else 0)
                d.append(j if chain or j == 0 else d[up] + 1)
            seen += bits
            depth += d
        lane_of = np.repeat(np.arange(n), counts)
        positions = context.repeat_interleave(i32(counts)) + i32(depth)
        tables = self.tables[:n]
        q = vi.norm_rotate_append(q, k, v, self.pool[0, 0], self.pool[0, 1], tables, i32(offsets), context, layer.cos,
                                  layer.sin, positions=positions, q_weight=layer.q_weight, k_weight=layer.k_weight)
        longest = int((context + i32(counts)).max())
        group = {} if only else dict(group_offsets=i32([0, n]), prefix_lens=i32([self.shared]), max_group_rows=sum(counts),
                                     max_prefix=self.shared)
        y = vi.prefix_attention(q, self.pool[0, 0], self.pool[0, 1], tables, i32(offsets), context, max_rows=max(counts),
                                max_own=longest - (0 if only else self.shared),
                                tree=None if chain else torch.tensor(seen, dtype=torch.int64, device=dev), **group)
        logits = (x + y.reshape(len(flat), -1) @ layer.out.T) @ layer.head.T
        # each row's drafted ancestors are history that the lane's state does not have yet
        extra, ends = [], [0]
        for t, p in zip(tokens, parents):
            for j in range(len(t)):
                up = j
                while not chain and up != 0:
                    extra.append(t[up])
                    up = p[up]
                ends.append(len(extra))
        logits = vi.process_logits(
            logits, self.params, lanes=i32(lane_of), state=self.state, extra=i32(extra),
            extra_offsets=torch.tensor(ends, dtype=torch.int64, device=dev), masks=self.masks,
            mask_index=flat % ALLOWED_EVERY, out=logits)
        return vi.greedy_packet(logits)["token"], context

    def round(self, anchors: list[int], drafts: list[list[int]], siblings: list[list[tuple[int, int]]]) -> list[list[int]]:
        """One speculative round: per lane the last token, a drafted chain and sibling leaves (depth, token) beside
        it.  Returns the tokens that each lane commits (the accepted path's, and the token that follows it)."""
        tokens = [[a, *d, *(t for _, t in s)] for a, d, s in zip(anchors, drafts, siblings)]
        parents = [[0, *range(len(d)), *(depth for depth, _ in s)] for d, s in zip(drafts, siblings)]
        picks, context = self.rows(tokens, parents)
        out, paths, at = [], [], 0
        for t, d, s in zip(tokens, drafts, siblings):
            mine = picks[at:at + len(t)].tolist()
            at += len(t)
            path, done = [0], [mine[0]]
            while len(path) <= len(d) and d[len(path) - 1] == done[-1]:     # the chain as far as it agrees
                path.append(len(path))
                done.append(mine[path[-1]])
            for i, (depth, token) in enumerate(s):                          # a sibling leaf that the target chose
                if depth == len(path) - 1 and token == done[-1]:
                    path.append(1 + len(d) + i)
                    done.append(mine[path[-1]])
                    break
            out.append(done)
            paths.append(path)
        i32 = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=self.device)  # noqa: E731
        width, kept = max(map(len, paths)), i32([len(p) for p in paths])
        vi.keep_rows(self.pool, self.tables, self.ids, context, i32([p + [0] * (width - len(p)) for p in paths]), kept)
        vi.pages_truncate(self.refs, self.tables, self.lengths, self.ids, context + kept, PAGE, self.status)
        self.state.update(i32([x for d in out for x in d]),
                          torch.tensor(np.concatenate([[0], np.cumsum([len(d) for d in out])]), device=self.device))
        assert not int(self.status[0]), "the pool has too few free pages"
        return out


def decode(lanes: Lanes, rounds: int, draft, anchors: list[int]) -> list[list[int]]:
    """Committed tokens per lane after some rounds; draft(lane, tokens) -> (chain, siblings)."""
    done = [[a] for a in anchors]
    for _ in range(rounds):
        plans = [draft(i, t) for i, t in enumerate(done)]
        for t, new in zip(done, lanes.round([t[-1] for t in done], [c for c, _ in plans], [s for _, s in plans])):
            t += new
    return done


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--lanes", type=int, default=4)
    ap.add_argument("--rounds", type=int, default=6)
    ap.add_argument("--seed", type=int, default=1)
    args = ap.parse_args()
    dev = torch.device("cuda:0")
    assert vi.load().vi_init() == 0, "device is not gfx950"
    rng = np.random.default_rng(args.seed)
    layer = Layer(args.seed, dev)
    prompt, anchors = rng.integers(0, VOCAB, 100).tolist(), rng.integers(0, VOCAB, args.lanes).tolist()
    plain = decode(Lanes(layer, args.lanes, prompt, dev), 5 * args.rounds, lambda lane, t: ([], []), anchors)

    def draft(lane, t):
        """A drafter that is right about the next tokens three times of four: what it proposes wrongly stands
        beside the right token as a sibling."""
        chain, sib = [], []
        for d in range(4):
            if len(t) + d >= len(plain[lane]):
                break
            right, wrong = plain[lane][len(t) + d], int(rng.integers(VOCAB))
            ok = rng.random() < 0.75
            chain.append(right if ok else wrong)
            if not ok:
                sib.append((d, right))
                break
        return chain, sib

    spec = decode(Lanes(layer, args.lanes, prompt, dev), args.rounds, draft, anchors)
    for i, (a, b) in enumerate(zip(plain, spec)):
        same = sum(x == y for x, y in zip(a, b))
        print(f"lane {i}: {len(b) - 1} tokens in {args.rounds} rounds ({(len(b) - 1) / args.rounds:.2f} a round), "
              f"{same} of {len(b)} as decoded one by one: {b[:12]}")


if __name__ == "__main__":
    main()
