"""Log probabilities of given tokens: texts are taken through the engine's step function in portions, as prompts
are, and every portion's logits give the next token's log probability, its rank, the entropy of the distribution it was
chosen from and the most likely alternatives (``kernels.token_logprobs``), without the logits leaving the GPU.

The reference's nearest thing is the teacher-forced loop of evaluate_int8_kv.py:74-90, which feeds
given tokens one by one and compares what a quantized cache makes of them.
"""

from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import torch

from ..ops import kernels
from .engine import StepEntry

# tokens of one step: their logits rows are kept on the GPU (512 of 50,257 are 103 MB)
PORTION = 512


@dataclass
class TokenScores:
    """Per token of a text; the first one has nothing in front of it."""

    token_ids: List[int]
    logprobs: List[Optional[float]]      # of each token given those in front of it (None for the first)
    ranks: List[Optional[int]]           # how many tokens were more likely
    entropies: List[Optional[float]]     # of the distribution that the token was taken from
    # with ``top``: the most likely tokens in its place, (token, log probability), the most likely first
    alternatives: Optional[List[Optional[List[Tuple[int, float]]]]] = None

    @property
    def total(self) -> float:
        """Log probability of the text given its first token."""
        return sum(value for value in self.logprobs if value is not None)


class _Rows:
    """What a portion's logits rows come to, on the GPU."""

    def __init__(self, rows: int, top: int, device):
        self.tokens = torch.empty(rows, dtype=torch.int32, device=device)
        self.floats = torch.empty((2, rows), dtype=torch.float32, device=device)
        self.ranks = torch.empty(rows, dtype=torch.int32, device=device)
        self.top_ids = torch.empty(rows * top, dtype=torch.int32, device=device) if top else None
        self.top_logprobs = torch.empty(rows * top, dtype=torch.float32, device=device) if top else None
        self.top = top
        self.partial = None

    def score(self, logits: torch.Tensor, tokens: Sequence[int]):
        """(log probabilities, entropies, ranks, alternatives) on the host."""
        rows, top = logits.shape[0], self.top
        self.tokens[:rows].copy_(torch.tensor(tokens, dtype=torch.int32))
        needed = kernels.logprob_scratch(rows, logits.shape[1], top)
        if needed and (self.partial is None or self.partial.numel() < needed):
            self.partial = torch.empty(needed, dtype=torch.float32, device=logits.device)
        ids = self.top_ids[:rows * top].view(rows, top) if top else None
        best = self.top_logprobs[:rows * top].view(rows, top) if top else None
        with torch.cuda.device_of(logits):         # (the engine's, which need not be the current one)
            kernels.token_logprobs(logits, self.tokens[:rows], self.floats[0, :rows], self.floats[1, :rows], self.ranks[:rows],
                                   ids, best, self.partial)
        alternatives = [None] * rows
        if top:
            alternatives = [list(zip(*pair)) for pair in zip(ids.tolist(), best.tolist())]
        return (*self.floats[:, :rows].tolist(), self.ranks[:rows].tolist(), alternatives)


def score_tokens(engine, texts: Sequence[Sequence[int]], top: int = 0) -> List[TokenScores]:
    """Scores of every text.  Short texts share a step; a long one goes through several.  The engine's requests that
    are live stay as they are; these take slots and pages beside them and give them back."""
    top = int(top)
    if not 0 <= top <= min(kernels.MAX_TOP, engine.spec.vocab_size):
        raise ValueError(f"0 to {min(kernels.MAX_TOP, engine.spec.vocab_size)} alternatives, not {top}")
    found = []
    for text in texts:
        tokens = [int(token) for token in text]
        if not tokens:
            raise ValueError("a text to be scored needs a token")
        if len(tokens) > engine.max_positions:
            raise ValueError(f"a text of {len(tokens)} tokens; the engine takes {engine.max_positions}")
        found.append(TokenScores(tokens, [None], [None], [None], [None] if top else None))
    budget = min(PORTION, engine.max_step_tokens)
    rows = _Rows(budget, top, engine.device)
    waiting = list(range(len(found)))
    live = {}                                  # text -> tokens that the engine has
    try:
        while waiting or live:
            entries, owners, room = [], [], budget
            for index in list(live):
                count = min(room, len(found[index].token_ids) - live[index])
                if count:
                    entries.append((index, count))
                    room -= count
            # a text joins a step that it fits whole, or one that it has for itself
            while waiting and room and (not entries or len(found[waiting[0]].token_ids) <= room) and _fits(
                    engine, found, entries, live, waiting[0]):
                index = waiting.pop(0)
                live[index] = 0
                count = min(room, len(found[index].token_ids))
                entries.append((index, count))
                room -= count
            if not entries:
                raise RuntimeError(f"no pages or slots are left for a text of {len(found[waiting[0]].token_ids)} tokens")
            step, following = [], []
            for index, count in entries:
                tokens, at = found[index].token_ids, live[index]
                # (the last token's row predicts nothing that is given)
                wanted = min(count, len(tokens) - at - 1)
                step.append(StepEntry(_request(index), tokens[at:at + count], list(range(wanted))))
                following += tokens[at + 1:at + 1 + wanted]
                owners += [index] * wanted
            output = engine.step(step)
            if following:
                for owner, logprob, entropy, rank, best in zip(owners, *rows.score(output.logits[:len(following)], following)):
                    text = found[owner]
                    text.logprobs.append(logprob)
                    text.entropies.append(entropy)
                    text.ranks.append(rank)
                    if top:
                        text.alternatives.append(best)
            for index, count in entries:
                live[index] += count
                if live[index] == len(found[index].token_ids):
                    del live[index]
                    engine.finish(_request(index))
    finally:
        for index in live:
            if engine.is_live(_request(index)):
                engine.finish(_request(index))
    return found


def _request(index: int):
    return ("score", index)


def _fits(engine, found, entries, live, index) -> bool:
    """Whether a slot, and pages for the whole of a text, are left beside those that are taken in already."""
    cache = engine.cache
    new = [at for at, _ in entries if not engine.is_live(_request(at))] + [index]
    if len(new) > len(cache.free_slots) or len(cache.requests) + len(new) > engine.max_requests:
        return False
    for group in range(len(cache.groups)):
        needed = sum(cache.pages_for_length(group, len(found[at].token_ids), PORTION)
                     for at in set(new) | set(live)) - sum(
            len([page for page in cache.requests[_request(at)].tables[group] if page >= 0])
            for at in live if engine.is_live(_request(at)))
        if needed > cache.pools[group].num_free:
            return False
    return True
