"""``PagedBackend`` on the GPU: the reference's paged backend
(src/server/backend/paged.py:21-99) over this package's ``TorchModel``.

Same batch composition (every generating sequence's next token first, then
prompt chunks under the ``prefill_chunk`` token budget, in sequence order),
same outputs (one ``StepOutput`` per sequence whose prompt is fully consumed),
same release rules.  The greedy argmax runs on the device and the step returns
after one copy of B token ids.

Tokenization is not on the attention path: the reference takes it from a GGUF
vocabulary through llama.cpp.  This backend takes any object with
``tokenize``, ``detokenize`` and ``is_end_of_generation``; without one it works
on token ids only (``QwenIds``: Qwen2.5's end-of-generation ids, no text).
"""

from __future__ import annotations

from collections import deque
from dataclasses import dataclass
from itertools import count

import torch

from .serve import BlockBudget
from .torch_model import PagedKVCache, PagedKVPool, TorchModel


@dataclass(frozen=True)
class StepOutput:
    """src/server/backend/base.py:5-8."""

    token: int
    finished: bool


class QwenIds:
    """Token-id-only vocabulary: <|endoftext|> (151643) and <|im_end|> (151645)
    end generation, as in Qwen2.5's vocabulary."""

    END_OF_GENERATION = frozenset({151643, 151645})

    def tokenize(self, text: str) -> list[int]:
        raise RuntimeError("no text vocabulary is attached; pass token ids")

    def detokenize(self, tokens: list[int]) -> bytes:
        raise RuntimeError("no text vocabulary is attached")

    def is_end_of_generation(self, token: int) -> bool:
        return token in self.END_OF_GENERATION


@dataclass
class _Sequence:
    cache: PagedKVCache
    pending: deque
    next_token: int | None = None  # the input of the next step, as an id or a token reference
    finished: bool = False
    feeds: object = None  # the launched step whose output the reference in next_token names


@dataclass
class LaunchedStep:
    """A step on the device: ``PagedBackend.finish`` turns it into outputs."""

    ids: object  # PendingTokens
    rows: list  # (seq_id, _Sequence, output row or None) per batch row


class PagedBackend:
    """src/server/backend/paged.py:21-99 with the model and pool on one GPU.

    ``num_blocks`` / ``block_size`` / ``prefill_chunk`` mean what they mean in
    the reference; ``max_seqs`` bounds the live sequences (device table rows).

    With a sliding window a sequence holds only the blocks it still sees
    (``sequence_blocks``) and may grow past the pool, up to the model's
    ``max_position`` tokens: a table row keeps an entry for every block a sequence
    ever had.  ``block_budget()`` admits requests by what they hold.

    ``pool_dtype`` torch.uint8 keeps the cache in 4 bits (3.5 times the tokens of bf16 in the
    same memory).
    """

    def __init__(self, model: TorchModel, num_blocks: int, block_size: int, prefill_chunk: int,
                 vocab=None, max_seqs: int = 256, pool_dtype: torch.dtype | None = None):
        self._model = model
        max_blocks = -(-model.max_position // block_size)
        if not model.config.attention_window:
            max_blocks = min(num_blocks, max_blocks)
        self._max_blocks = max_blocks
        self._pool = PagedKVPool(model.config, num_blocks, block_size, device=model.device,
                                 dtype=pool_dtype or model.dtype, max_seqs=max_seqs,
                                 max_blocks_per_seq=max_blocks)
        self._num_blocks = num_blocks
        self._prefill_chunk = prefill_chunk
        self._vocab = vocab if vocab is not None else QwenIds()
        self._ids = count()
        self._sequences: dict[int, _Sequence] = {}

    @property
    def blocks_in_use(self) -> int:
        return self._num_blocks - self._pool.free_blocks

    @property
    def pool(self) -> PagedKVPool:
        return self._pool

    @property
    def sequence_blocks(self) -> int | None:
        """The most blocks that a sequence holds at a time (None: as many as its tokens fill).

        While a step adds n <= prefill_chunk tokens to L cached ones, these are the
        sinks' and those of tokens L - window + 1 to L + n - 1, which begin anywhere in
        their first block."""
        config, size = self._model.config, self._pool.block_size
        if not config.attention_window:
            return None
        seen = config.attention_window - 1 + max(self._prefill_chunk, 1)
        return -(-config.attention_sinks // size) + (seen + 2 * size - 2) // size

    def block_budget(self) -> BlockBudget:
        """The admission budget of this backend's pool."""
        return BlockBudget(self._num_blocks, self._pool.block_size, self.sequence_blocks,
                           self._max_blocks * self._pool.block_size)

    def tokenize(self, text: str) -> list[int]:
        return self._vocab.tokenize(text)

    def detokenize(self, tokens: list[int]) -> bytes:
        return self._vocab.detokenize(tokens)

    def start_sequence(self, prompt_tokens: list[int]) -> int:
        seq_id = next(self._ids)
        cache = self._pool.new_cache(seq_id)
        cache.reserve(0)
        self._sequences[seq_id] = _Sequence(cache, deque(prompt_tokens))
        return seq_id

    def fork_sequence(self, seq_id: int, prompt_tokens: list[int]) -> int:
        """Starts a sequence that continues seq_id's tokens so far with
        ``prompt_tokens`` (a shared prompt, another turn of a conversation): what
        is cached for seq_id is shared, not computed again.  Without
        ``prompt_tokens`` the new sequence generates what seq_id would.  A step
        that seq_id still runs in must be finished first."""
        parent = self._sequences[seq_id]
        if parent.feeds is not None:
            raise RuntimeError(f"sequence {seq_id} has an unfinished step")
        if parent.finished and not prompt_tokens:
            raise RuntimeError(f"sequence {seq_id} has finished: a fork needs new tokens")
        child_id = next(self._ids)
        child = _Sequence(self._pool.fork(parent.cache, child_id), deque(parent.pending))
        if parent.next_token is not None:
            if prompt_tokens:
                child.pending.append(parent.next_token)
            else:
                child.next_token = parent.next_token
        child.pending.extend(prompt_tokens)
        self._sequences[child_id] = child
        return child_id

    def compact(self) -> int:
        """Moves the cache blocks in use to the lowest ids; returns how many moved."""
        return self._pool.compact()

    def step(self) -> dict[int, StepOutput]:
        launched = self.launch()
        return self.finish(launched) if launched is not None else {}

    def launch(self) -> LaunchedStep | None:
        """Composes and launches one step without waiting for it (the batch of
        ``step``).  A generating sequence whose last token has not reached the
        host yet feeds it by reference from the device, so the next step can be
        composed while this one runs; ``finish`` returns this step's outputs.
        A sequence that ends on an end-of-generation token revealed only by
        ``finish`` of the previous step still runs in this one: that row's
        output is dropped (``finish`` skips finished sequences)."""
        batch = self._generating_inputs() + self._prefill_inputs()
        if not batch:
            return None
        pending = self._model.launch_tokens(
            [(toks, self._sequences[s].cache) for s, toks in batch])
        rows = []
        for row, (seq_id, _) in enumerate(batch):
            sequence = self._sequences[seq_id]
            if sequence.pending:
                rows.append((seq_id, sequence, None))
            else:
                rows.append((seq_id, sequence, row))
        launched = LaunchedStep(pending, rows)
        for seq_id, sequence, row in rows:
            if row is not None:
                sequence.next_token = pending.ref(row)  # resolved on the device
                sequence.feeds = launched
        return launched

    def finish(self, launched: LaunchedStep) -> dict[int, StepOutput]:
        """Waits for a launched step: {seq_id: StepOutput} for every sequence
        whose prompt was fully consumed and that had not finished before."""
        tokens = launched.ids.result()
        outputs = {}
        for seq_id, sequence, row in launched.rows:
            if row is None or sequence.finished:
                if sequence.feeds is launched:
                    # The row that ran on past the end: its input, the ending token, is
                    # cached, and its output is nobody's.
                    sequence.next_token = sequence.feeds = None
                continue
            token = tokens[row]
            if sequence.feeds is launched:
                sequence.next_token = token  # not relaunched yet: feed the id itself
                sequence.feeds = None
            sequence.finished = self._vocab.is_end_of_generation(token)
            outputs[seq_id] = StepOutput(token, sequence.finished)
        return outputs

    def draft_step(self, drafts: dict[int, list[int]], temperature: float = 0.0,
                   generator: torch.Generator | None = None) -> dict[int, list[StepOutput]]:
        """One step of the generating sequences with drafted tokens: verifies ``drafts[seq_id]``
        (looked up in the text, or a small model's most likely tokens), the tokens that may
        follow seq_id's last one, and returns each sequence's outputs: the drafts that hold
        and the token after them, up to one that ends the generation.  A sequence without
        drafts gives one output, as in ``step``.  With temperature 0 the outputs are
        ``step``'s; else they are distributed as the model's samples at that temperature,
        by random numbers from ``generator`` (on the model's device).  Prompts wait for
        ``step``; a launched step must be finished first.

        Drafts behind one that would end the generation are not looked at, nor are those past
        the last position, or for whose tokens no block is free once every sequence has one
        for its next token: a step that runs without drafts runs with them, and behind it a
        sequence holds the blocks of its cached tokens, as after plain steps.  What a request
        may still generate is the caller's to know: outputs past that count against the pool."""
        batch = []
        for seq_id, tokens in self._generating_inputs():
            if self._sequences[seq_id].feeds is not None:
                raise RuntimeError(f"sequence {seq_id} has an unfinished step")
            batch.append((seq_id, tokens + self._up_to_end(drafts.get(seq_id, ()))))
        if not batch:
            return {}
        batch = self._with_room(batch)
        uniforms = None
        if temperature != 0.0:
            uniforms = torch.rand(sum(len(tokens) for _, tokens in batch), generator=generator,
                                  device=self._model.device)
        results = self._model.verify_tokens(
            [(tokens, self._sequences[s].cache) for s, tokens in batch], temperature, uniforms)
        outputs = {}
        for (seq_id, _), tokens in zip(batch, results):
            sequence = self._sequences[seq_id]
            sequence.next_token = tokens[-1]
            # Of the drafts that hold only the last may end the generation.  It is cached then:
            # the token behind it is nobody's, and a fork has nothing to feed again.
            if len(tokens) > 1 and self._vocab.is_end_of_generation(tokens[-2]):
                tokens, sequence.next_token = tokens[:-1], None
            sequence.finished = self._vocab.is_end_of_generation(tokens[-1])
            outputs[seq_id] = [StepOutput(token, False) for token in tokens[:-1]]
            outputs[seq_id].append(StepOutput(tokens[-1], sequence.finished))
        return outputs

    def release_sequence(self, seq_id: int) -> None:
        self._pool.release(self._sequences.pop(seq_id).cache)

    def close(self) -> None:
        pass

    def _up_to_end(self, drafts) -> list[int]:
        """Drafts as far as the first that would end the generation."""
        tokens = []
        for token in drafts:
            tokens.append(token)
            if self._vocab.is_end_of_generation(token):
                break
        return tokens

    def _with_room(self, batch) -> list[tuple[int, list[int]]]:
        """The batch with as many drafts of each sequence, in turn, as positions and blocks are
        left for."""
        pool, size = self._pool, self._pool.block_size
        last = min(self._model.max_position, self._max_blocks * size)
        lengths = [self._sequences[s].cache.length for s, _ in batch]
        own = [max(pool.allocator.held_blocks(s), -(-(n + 1) // size))
               for (s, _), n in zip(batch, lengths)]  # blocks, the next token's with them
        free = pool.free_blocks - sum(
            n - pool.allocator.held_blocks(s) for (s, _), n in zip(batch, own))
        cut = []
        for (seq_id, tokens), length, blocks in zip(batch, lengths, own):
            room = min(last, (blocks + max(free, 0)) * size) - length
            tokens = tokens[: max(room, 1)]
            free -= max(0, -(-(length + len(tokens)) // size) - blocks)
            cut.append((seq_id, tokens))
        return cut

    def _generating_inputs(self) -> list[tuple[int, list[int]]]:
        return [
            (seq_id, [sequence.next_token])
            for seq_id, sequence in self._sequences.items()
            if not sequence.pending and not sequence.finished
        ]

    def _prefill_inputs(self) -> list[tuple[int, list[int]]]:
        inputs = []
        remaining = self._prefill_chunk
        for seq_id, sequence in self._sequences.items():
            take = min(remaining, len(sequence.pending))
            if take:
                inputs.append((seq_id, [sequence.pending.popleft() for _ in range(take)]))
                remaining -= take
        return inputs
