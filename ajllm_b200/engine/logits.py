"""Penalties, token biases and token masks of a batch of requests, applied to its logits before sampling.

What a request's penalties look at (its prompt and its output) stays in device memory between steps: a step uploads
only the tokens that are new since the request's previous one, and the rows of the batch are gathered on the device.
"""

from __future__ import annotations

import torch

from ajllm_b200.engine.scheduler import SamplingParams, Sequence
from ajllm_b200.ops import serving

_LARGEST = 1e6            # of a bias or penalty: far above any logit, far below what overflows fp32 when it adds up


def check_params(params: SamplingParams, vocab_size: int) -> None:
    """Raises ``ValueError`` for values that :class:`LogitsProcessor` cannot apply."""
    if not 1.0 / _LARGEST <= params.repetition_penalty <= _LARGEST:
        raise ValueError(f"repetition_penalty must be positive, between {1 / _LARGEST:g} and {_LARGEST:g} (got {params.repetition_penalty})")
    for name in ("presence_penalty", "frequency_penalty"):
        value = getattr(params, name)
        if not -_LARGEST <= value <= _LARGEST:
            raise ValueError(f"{name} must be a number of at most {_LARGEST:g} (got {value})")
    for token, value in (params.logit_bias or {}).items():
        if not 0 <= int(token) < vocab_size:
            raise ValueError(f"logit_bias: token {token} is not in the vocabulary of {vocab_size}")
        if not -_LARGEST <= value <= _LARGEST:
            raise ValueError(f"logit_bias: the bias of token {token} must be a number of at most {_LARGEST:g} (got {value})")
    if params.token_mask is not None and not callable(params.token_mask):
        raise ValueError("token_mask must be callable: output tokens -> int32 words of allowed tokens, or None")


class LogitsProcessor:
    """``masks`` asks the requests of a batch which tokens may follow, ``apply`` returns the batch's processed logits, and
    ``forget`` drops what is held for a finished request."""

    def __init__(self, vocab_size: int, device: torch.device) -> None:
        self.vocab_size, self.device = vocab_size, device
        self.words = (vocab_size + 31) // 32
        self._history = torch.zeros(0, 0, dtype=torch.int32, device=device)      # [slots, longest sequence so far]
        self._slots: dict[int, int] = {}           # request -> its row of the history
        self._filled: dict[int, int] = {}          # request -> tokens of it that are in the row
        self._free: list[int] = []
        self._key: tuple[int, ...] | None = None   # the batch that the tensors below belong to
        self._batch: dict[str, torch.Tensor | None] = {}

    def forget(self, request_id: int) -> None:
        slot = self._slots.pop(request_id, None)
        if slot is not None:
            del self._filled[request_id]
            self._free.append(slot)

    def apply(self, seqs: list[Sequence], logits: torch.Tensor, mask: torch.Tensor | None = None) -> torch.Tensor:
        """The logits to sample a token of ``seqs[i]`` from in row ``i``; ``mask`` comes from :meth:`masks`."""
        if not any(s.params.processes_logits for s in seqs):
            return logits
        key = tuple(s.request_id for s in seqs)
        if key != self._key:
            self._key, self._batch = None, self._per_request([s.params for s in seqs])
            self._key = key
        penalties = {}
        if any(s.params.penalises for s in seqs):
            penalties = dict(zip(("history", "prompt_lens", "history_lens"), self._histories(seqs)))
            penalties.update((name, self._batch[name]) for name in ("repetition", "presence", "frequency"))
        return serving.process_logits(logits, **penalties, bias_ids=self._batch["bias_ids"],
                                      bias_values=self._batch["bias_values"], token_mask=mask)

    def _per_request(self, params: list[SamplingParams]) -> dict[str, torch.Tensor | None]:
        def column(values: list[float], neutral: float) -> torch.Tensor | None:
            if all(v == neutral for v in values):
                return None
            return torch.tensor(values, dtype=torch.float32, device=self.device)

        batch = {"repetition": column([p.repetition_penalty for p in params], 1.0),
                 "presence": column([p.presence_penalty for p in params], 0.0),
                 "frequency": column([p.frequency_penalty for p in params], 0.0), "bias_ids": None, "bias_values": None}
        widest = max(len(p.logit_bias or {}) for p in params)
        if widest:
            biases = [list((p.logit_bias or {}).items()) for p in params]
            batch["bias_ids"] = torch.tensor([[int(t) for t, _ in row] + [-1] * (widest - len(row)) for row in biases],
                                             dtype=torch.int32, device=self.device)
            batch["bias_values"] = torch.tensor([[float(v) for _, v in row] + [0.0] * (widest - len(row)) for row in biases],
                                                dtype=torch.float32, device=self.device)
        return batch

    def _histories(self, seqs: list[Sequence]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """History rows of the batch, their prompt lengths and their lengths; a request without penalties has length 0."""
        for seq in seqs:
            if seq.params.penalises and seq.request_id not in self._slots:
                self._slots[seq.request_id] = self._free.pop() if self._free else len(self._slots)
                self._filled[seq.request_id] = 0
        longest = max(s.total_len for s in seqs if s.params.penalises)
        rows, width = self._history.shape
        if len(self._slots) + len(self._free) > rows or longest > width:
            grown = torch.zeros(max(rows, 2 * (len(self._slots) + len(self._free))), max(width, 2 * longest), dtype=torch.int32,
                                device=self.device)
            grown[:rows, :width] = self._history
            self._history = grown
        rows, width = self._history.shape
        places, tokens, slots, prompts, totals = [], [], [], [], []
        for seq in seqs:
            if not seq.params.penalises:
                slots.append(0)
                prompts.append(0)
                totals.append(0)
                continue
            slot, have, total = self._slots[seq.request_id], self._filled[seq.request_id], seq.total_len
            places.extend(range(slot * width + have, slot * width + total))
            tokens.extend(seq.token_slice(have, total))
            self._filled[seq.request_id] = total
            slots.append(slot)
            prompts.append(len(seq.prompt))
            totals.append(total)
        n, new = len(seqs), len(tokens)
        packed = torch.tensor(slots + prompts + totals + places + tokens, dtype=torch.long, device=self.device)
        if new:
            self._history.view(-1).index_copy_(0, packed[3 * n:3 * n + new], packed[3 * n + new:].int())
        lens = packed[n:3 * n].int()
        return self._history[:, :longest].index_select(0, packed[:n]), lens[:n], lens[n:]

    def masks(self, seqs: list[Sequence]) -> tuple[torch.Tensor | None, list[bool]]:
        """Mask words of every row (``None``: no request has a mask), and whether the row's mask leaves no token (such a
        row is left unmasked: its request has to end)."""
        emptied = [False] * len(seqs)
        if not any(s.params.token_mask is not None for s in seqs):
            return None, emptied
        mask = torch.full((len(seqs), self.words), -1, dtype=torch.int32)
        tail = (1 << (self.vocab_size - 32 * (self.words - 1))) - 1        # bits of the last word that are tokens
        for i, seq in enumerate(seqs):
            words = seq.params.token_mask(list(seq.output)) if seq.params.token_mask is not None else None
            if words is None:
                continue
            words = torch.as_tensor(words)
            if words.dtype != torch.int32 or words.shape != (self.words,):
                raise ValueError(f"token_mask must return int32 words [{self.words}], one bit per token (got {words.dtype} {tuple(words.shape)})")
            words = words.cpu()
            emptied[i] = not (bool(words[:-1].any()) or int(words[-1]) & tail)
            if not emptied[i]:
                mask[i] = words
        return mask.to(self.device), emptied
