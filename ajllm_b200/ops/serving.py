"""GPU entry points of the serving path: in-place RoPE on packed rows with explicit positions, paged
attention for decode / verify rows, the training flash kernel for prompts that start from an empty
cache, and the batched sampler; block tables and slot maps built on the device, paged attention of a batch
behind a shared prefix, and logits processing (these three take CPU tensors too and then run the plain
statements of :mod:`ajllm_b200.ops.reference`)."""

from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch

from ajllm_b200.ops import native, reference

_MAX_ROWS = 64


def rope_packed_(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, num_heads: int,
                 num_kv_heads: int, head_dim: int) -> None:
    """Rotate the q and k heads of packed ``[tokens, (Hq + 2 Hkv) * hd]`` rows in place at ``positions``."""
    native.call("ajb_rope_qk", qkv.data_ptr(), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), qkv.shape[0], 1,
                num_heads, num_kv_heads, head_dim, qkv.stride(0), 0, native.stream_ptr())


class PagedPlan:
    """Launch plan of one ragged decode / verify batch: sequences grouped by their number of new rows, with the
    block tables, row offsets and context lengths of every group already on the device. Built once per engine
    step and reused by every layer."""

    def __init__(self, block_tables: torch.Tensor, q_lens_host: list[int], context_lens_host: list[int], heads: int,
                 kv_heads: int) -> None:
        group = heads // kv_heads
        max_q = max(1, _MAX_ROWS // group)
        classes: dict[int, list[tuple[int, int, int]]] = {}
        cursor = 0
        for i, (n, ctx) in enumerate(zip(q_lens_host, context_lens_host)):
            for a in range(0, n, max_q):
                b = min(n, a + max_q)
                classes.setdefault(b - a, []).append((i, cursor + a, ctx - (n - b)))
            cursor += n
        self.total_rows = cursor
        self.max_context = max(context_lens_host) if context_lens_host else 0
        device = block_tables.device
        self.launches = []
        identity = list(range(block_tables.shape[0]))
        for q_len, items in classes.items():
            rows = [it[0] for it in items]
            tables = block_tables if rows == identity else \
                block_tables.index_select(0, torch.tensor(rows, dtype=torch.long, device=device)).contiguous()
            packed = torch.tensor([[it[1] for it in items], [it[2] for it in items]], dtype=torch.int32, device=device)
            self.launches.append((q_len, len(items), tables, packed[0], packed[1]))


def paged_attention_planned(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, plan: PagedPlan,
                            scale: float | None = None) -> torch.Tensor:
    """``scale`` defaults to ``1 / sqrt(head width of q)``; callers whose heads are zero-padded pass the true one."""
    total, heads, head_dim = q.shape
    kv_heads = key_cache.shape[2]
    out = torch.empty_like(q)
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    num_blocks, block_size = key_cache.shape[0], key_cache.shape[1]
    for q_len, count, tables, starts, ctxs in plan.launches:
        # few (sequence, KV head) pairs cannot fill the device: cut every sequence's keys over several CTAs, up to
        # two CTAs per SM (what the kernel's shared memory admits) and never more parts than the longest context has
        # 64-key tiles
        max_context = getattr(plan, "max_context", None) or tables.shape[1] * block_size
        splits = paged_splits(count * kv_heads, max_context, heads // kv_heads * q_len, head_dim)
        part_o = part_ml = None
        if splits > 1:
            part_o = torch.empty(total, heads, splits, head_dim, dtype=torch.float32, device=q.device)
            part_ml = torch.empty(total, heads, splits, 2, dtype=torch.float32, device=q.device)
        native.call("ajb_paged_attention", q.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), tables.data_ptr(),
                    ctxs.data_ptr(), starts.data_ptr(), out.data_ptr(), count, num_blocks, block_size,
                    tables.shape[1], heads, kv_heads, head_dim, q_len, scale, splits, native.ptr(part_o),
                    native.ptr(part_ml), native.stream_ptr())
    return out


_SM_COUNT: list[int] = []


def paged_splits(ctas: int, max_context: int, rows: int = 1, head_dim: int = 128) -> int:
    """Parts per sequence for the paged-attention kernels given the (sequence, KV head) pairs of a launch, the query rows of a
    pair and the width of its heads."""
    if not _SM_COUNT:
        _SM_COUNT.append(int(native.lib().ajb_sm_count()))
    # One each for nearly all SMs. Up to 32 rows of 128-wide heads, whose CTAs fill an SM's memory path, that is best: 128 pairs
    # x 4096 keys, 4 rows: 63.5 us whole and in two parts, 32 rows: 63.5 us whole, 67.6 us in two parts. Other CTAs want a second
    # one beside them: 64-wide heads, 8 rows: 45.1 and 38.9 us (16384 keys: 154 and 107 us), 40 rows of 128: 82.1 and 67.6 us.
    if 5 * ctas >= 4 * _SM_COUNT[0] and rows <= 32 and head_dim == 128:
        return 1
    want = (2 * _SM_COUNT[0]) // max(1, ctas)
    tiles = max(1, (max_context + 63) // 64)
    # a part should keep enough 64-key steps to amortise its start and the merge kernel: 16 steps when the launch
    # already covers half the SMs (measured: 16 sequences x 1024 keys, 24 us whole against 34 us in two parts), 8 below that
    per_part = 16 if 2 * ctas >= _SM_COUNT[0] else 8
    return max(1, min(want, tiles // per_part, 16))


def paged_attention(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
                    context_lens, q_lens, q_lens_host: list[int], context_lens_host: list[int]) -> torch.Tensor:
    """Ragged decode / verify attention. ``q`` is ``[total_rows, Hq, hd]``; launches are grouped by the
    number of new rows per sequence, and long row runs are cut into chunks the kernel can hold."""
    plan = PagedPlan(block_tables, q_lens_host, context_lens_host, q.shape[1], key_cache.shape[2])
    return paged_attention_planned(q, key_cache, value_cache, plan)


def prompt_attention(qkv_rows: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int,
                     scale: float | None = None) -> torch.Tensor:
    """Causal attention of one prompt that starts from an empty cache, read in place from its packed
    (already rotated) ``[T, (Hq + 2 Hkv) * hd]`` rows. Returns ``[T, Hq * hd]``."""
    T, width = qkv_rows.shape
    out = torch.empty(T, num_heads * head_dim, dtype=torch.bfloat16, device=qkv_rows.device)
    lse = torch.empty(num_heads, T, dtype=torch.float32, device=qkv_rows.device)
    native.call("ajb_flash_fwd", qkv_rows.data_ptr(), out.data_ptr(), lse.data_ptr(), 1, T, num_heads, num_kv_heads,
                head_dim, qkv_rows.stride(0), 1, 1.0 / math.sqrt(head_dim) if scale is None else scale,
                native.stream_ptr())
    return out


def sample_rows(logits: torch.Tensor, temperature: torch.Tensor, top_p: torch.Tensor, seeds: torch.Tensor,
                counters: torch.Tensor) -> torch.Tensor:
    """One token per row of fp32 ``logits`` ``[rows, vocab]``; per-row temperature (``<= 0`` = greedy),
    top-p, and a counter-based random stream ``(seed, counter)``. Returns int32 ``[rows]`` on the device."""
    logits = logits.contiguous()
    rows, vocab = logits.shape
    out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    # few rows over a large vocabulary: the row maxima are found by about two CTAs per SM, not one CTA per row
    if not _SM_COUNT:
        _SM_COUNT.append(int(native.lib().ajb_sm_count()))
    chunks = max(1, min(2 * _SM_COUNT[0] // max(1, rows), vocab // 4096, 64))
    workspace = torch.empty(rows, chunks, 2, dtype=torch.int32, device=logits.device) if chunks > 1 else None
    native.call("ajb_sample_rows", logits.data_ptr(), logits.stride(0), rows, vocab,
                temperature.data_ptr(), top_p.data_ptr(), seeds.data_ptr(), counters.data_ptr(), out.data_ptr(),
                chunks, native.ptr(workspace), native.stream_ptr())
    return out


def spec_verify(target_logits: torch.Tensor, draft_logits: torch.Tensor, draft_tokens: torch.Tensor,
                temperature: torch.Tensor, seeds: torch.Tensor, counters: torch.Tensor) -> torch.Tensor:
    """Accept/reject step of speculative decoding for a batch of sequences.

    ``target_logits [seqs, k + 1, vocab]``, ``draft_logits [seqs, k, vocab]`` (fp32), ``draft_tokens [seqs, k]``
    (int32). Returns int32 ``[seqs, 2]`` = (accepted draft tokens, next token)."""
    seqs, k1, vocab = target_logits.shape
    result = torch.empty(seqs, 2, dtype=torch.int32, device=target_logits.device)
    native.call("ajb_spec_verify", target_logits.contiguous().data_ptr(), draft_logits.contiguous().data_ptr(),
                draft_tokens.contiguous().data_ptr(), seqs, k1 - 1, vocab, temperature.data_ptr(), seeds.data_ptr(),
                counters.data_ptr(), result.data_ptr(), native.stream_ptr())
    return result


# ----------------------------------------------------------------------------- shared by the operators below


# A small operator takes a few microseconds on the device. Its ordinary call on a GPU is checked, allocated and launched by
# an extension (csrc/fast_calls.cpp), which leaves every other call to the code here. The argument checks are one expression
# over cheap attributes; only when it fails are the arguments gone through one by one for the message.
_I32, _I64, _F32, _BF16 = torch.int32, torch.int64, torch.float32, torch.bfloat16
_CONTIGUOUS = torch.contiguous_format


def _dense(op: str, name: str, t: torch.Tensor, dtype: torch.dtype, device: torch.device, shape: tuple[int, ...]) -> None:
    if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{op}: {name} must be a contiguous {dtype} tensor of shape {list(shape)} on {device} "
                         f"(got {t.dtype} {list(t.shape)} on {t.device}, strides {t.stride()})")


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory ranges that two non-empty tensors span have a byte in common."""
    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


# ----------------------------------------------------------------------------- block tables and slot maps


class BatchMaps(NamedTuple):
    """What the kernels of one serving step need to know about a ragged batch of ``n`` sequences."""

    tables: torch.Tensor          # int32 [n, max_blocks]: block ids of every sequence, padded
    positions: torch.Tensor       # int32 [total_tokens]: position of every new token in its sequence
    slots: torch.Tensor           # int64 [total_tokens]: cache slot of every new token
    q_start: torch.Tensor         # int32 [n + 1]: first row of every sequence, and the end of the last
    context_lens: torch.Tensor    # int32 [n]: cached plus new tokens


def batch_maps(block_ids: torch.Tensor, block_counts: torch.Tensor, cached_lens: torch.Tensor, q_lens: torch.Tensor,
               total_tokens: int, max_blocks: int, *, block_size: int = 16, pad_block: int = 0,
               out: "BatchMaps | tuple[torch.Tensor, ...] | None" = None) -> BatchMaps:
    """Block tables, positions, cache slots, row offsets and context lengths of a ragged batch, built on the device.

    ``block_ids`` holds the cache blocks of all sequences one after another, ``block_counts[i]`` of them for sequence
    ``i``, which has ``cached_lens[i]`` tokens in the cache and brings ``q_lens[i]`` new ones (any of them may be 0);
    all four are int32. ``total_tokens`` is the number of rows of the step: rows behind the last sequence, and tokens
    for which a sequence has no block, are sent to ``pad_block`` (the former to position 0 and the block's first slot),
    which must be a block that no sequence owns. Table rows keep a sequence's first ``max_blocks`` blocks and are filled
    up with ``pad_block``. At most 16384 sequences per call.

    ``out`` may hold the five result tensors (buffers a captured graph reads), apart from the inputs and from one another;
    they are overwritten and returned. On a GPU the first three start on 16-byte boundaries.
    """
    if native.fast is not None:
        found = native.fast.batch_maps(block_ids, block_counts, cached_lens, q_lens, total_tokens, max_blocks, block_size, pad_block, out)
        if found is not None:
            native.launch_count += 1
            return BatchMaps._make(out if found is True else found)
    index, each = block_ids.get_device(), block_counts.shape
    if not (block_ids.dtype is block_counts.dtype is cached_lens.dtype is q_lens.dtype is _I32
            and block_counts.get_device() == index == cached_lens.get_device() == q_lens.get_device()
            and block_ids.dim() == 1 and len(each) == 1 and cached_lens.shape == each == q_lens.shape
            and block_ids.is_contiguous() and block_counts.is_contiguous() and cached_lens.is_contiguous() and q_lens.is_contiguous()):
        if block_counts.dim() != 1 or block_ids.dim() != 1:
            raise ValueError("batch_maps: block_ids is one flat list, block_counts has one entry per sequence")
        for name, t, shape in (("block_ids", block_ids, block_ids.shape), ("block_counts", block_counts, each),
                               ("cached_lens", cached_lens, each), ("q_lens", q_lens, each)):
            _dense("batch_maps", name, t, _I32, block_ids.device, shape)
    n = each[0]
    if not (0 <= total_tokens < 1 << 30 and max_blocks >= 1 and block_size >= 1 and pad_block >= 0 and n <= 16384):
        raise ValueError(f"batch_maps: total_tokens {total_tokens} and pad_block {pad_block} must not be negative, max_blocks {max_blocks} "
                         f"and block_size {block_size} must be positive, and there are at most 16384 sequences (got {n})")
    if out is not None:
        tables, positions, slots, q_start, context_lens = out
        if not (tables.dtype is positions.dtype is q_start.dtype is context_lens.dtype is _I32 and slots.dtype is _I64
                and tables.get_device() == index == positions.get_device() == slots.get_device() == q_start.get_device() == context_lens.get_device()
                and tables.shape == (n, max_blocks) and positions.shape == (total_tokens,) == slots.shape and q_start.shape == (n + 1,)
                and context_lens.shape == each and tables.is_contiguous() and positions.is_contiguous() and slots.is_contiguous()
                and q_start.is_contiguous() and context_lens.is_contiguous()):
            for name, t, dtype, shape in (("tables", tables, _I32, (n, max_blocks)), ("positions", positions, _I32, (total_tokens,)),
                                          ("slots", slots, _I64, (total_tokens,)), ("q_start", q_start, _I32, (n + 1,)),
                                          ("context_lens", context_lens, _I32, each)):
                _dense("batch_maps", "out." + name, t, dtype, block_ids.device, shape)
    if index < 0:
        found = reference.batch_maps(block_ids, block_counts, cached_lens, q_lens, total_tokens, max_blocks, block_size, pad_block)
        if out is None:
            return BatchMaps(*found)
        if any(_overlap(a, b) for i, a in enumerate(out) for b in (*out[:i], block_ids, block_counts, cached_lens, q_lens)):
            raise ValueError("batch_maps: out must lie apart from the inputs and from one another")
        for mine, theirs in zip(out, found):
            mine.copy_(theirs)
        return BatchMaps(*out)
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return batch_maps(block_ids, block_counts, cached_lens, q_lens, total_tokens, max_blocks, block_size=block_size,
                              pad_block=pad_block, out=out)
    if out is None:
        device = block_ids.device
        tables, positions = torch.empty(n, max_blocks, dtype=_I32, device=device), torch.empty(total_tokens, dtype=_I32, device=device)
        slots = torch.empty(total_tokens, dtype=_I64, device=device)
        q_start, context_lens = torch.empty(n + 1, dtype=_I32, device=device), torch.empty(n, dtype=_I32, device=device)
    native.call_packed("ajb_batch_maps", block_ids.data_ptr(), block_counts.data_ptr(), cached_lens.data_ptr(), q_lens.data_ptr(),
                block_ids.shape[0], n, total_tokens, max_blocks, block_size, pad_block, tables.data_ptr(), positions.data_ptr(),
                slots.data_ptr(), q_start.data_ptr(), context_lens.data_ptr(), native.stream_ptr(index))
    return BatchMaps(tables, positions, slots, q_start, context_lens)


# ----------------------------------------------------------------------------- attention behind a shared prefix

_PREFIX_TILE = 128         # query rows and keys per step of the prefix kernel


@functools.lru_cache(maxsize=4096)
def prefix_plan(n: int, q_len: int, group: int, kv_heads: int, head_dim: int, shared: int, behind: int,
                known: int) -> tuple[int, int, int, int]:
    """How a call of :func:`shared_prefix_attention` is divided: ``(query tokens per piece of the prefix in the paged launch,
    or 0 for the prefix kernel; divisions of the prefix; divisions of a suffix; parts per row in all)``. Suffixes have at most
    ``behind`` tokens; unless that is ``known`` to be what they have, the division is the one that does best for suffixes of
    up to that and up to half of it together, or, in tables with room for more than 1024 behind the prefix, of up to 128 and
    up to 512 (such tables are often much wider than contexts: 64 sequences behind 2048 + 32 tokens in tables for 8192 took
    45 us when divided for the tables, 21 us now). Whichever of the two forms is
    estimated to end first is taken (in us, from measurements of 4 to 1024 query rows per KV head, prefixes of 512 to 7680
    and suffixes of 32 to 1024 tokens)."""
    if not _SM_COUNT:
        _SM_COUNT.append(int(native.lib().ajb_sm_count()))
    sms = _SM_COUNT[0]
    chunk = q_len if group * q_len <= 32 else max(1, min(q_len, _PREFIX_TILE // group))
    pieces = n * kv_heads * -(-q_len // chunk)
    if not shared:
        alone = paged_splits(pieces, behind, group * chunk, head_dim)
        return 0, 0, alone, alone
    # where the suffixes are not known to be long, they are divided as if alone, which costs little if they are short
    bound_splits = paged_splits(pieces, behind)
    tiles, most = -(-shared // _PREFIX_TILE), -(-behind // _PREFIX_TILE)
    divisions = tuple(range(1, min(16, max(1, most)) + 1)) if known or behind <= 1024 else (min(8, bound_splits),)
    rows = n * q_len * group
    times = []
    for expected in (behind,) if known else (behind // 2, behind) if behind <= 1024 else (128, 512):
        least = 3.0 + (n * expected + shared) * kv_heads * head_dim * 4 / 6.5e6       # reading the caches once
        found = _kernel_plans(n, rows, pieces, kv_heads, head_dim, tiles, expected, divisions, least, sms)
        if group * q_len <= 32:
            found.update(_pieces_plans(n, q_len, group, kv_heads, head_dim, tiles, expected, divisions, least, sms))
        times.append((min(found.values()), found))
    return min(times[0][1], key=lambda plan: (sum(found[plan] / best for best, found in times), plan))


def _pieces_plans(n, q_len, group, kv_heads, head_dim, tiles, expected, divisions, least, sms):
    """The prefix in pieces of the paged launch, for 16 query rows each (32 where a sequence has more than 16): a second read
    of the prefix from L2 costs less than pieces of 32 rows, of which an SM holds one instead of two (8 sequences of 4 rows,
    512 + 32 tokens: 7.2 us against 7.8). A piece takes 3 us and 1.1 us per 128 keys (32 rows: 1.5 us)."""
    height = 16 if group * q_len <= 16 else 32
    tokens = height // group
    slots = sms * (2 if height == 16 or head_dim == 64 else 1)
    step = 1.1 if height == 16 else 1.5
    units = kv_heads * -(-n * q_len // tokens)
    per_part = 0.1 + 0.0005 * n * q_len * group * kv_heads
    suffix_tiles = -(-expected // _PREFIX_TILE)
    found = {}
    for splits in divisions:
        back, back_time = n * kv_heads * max(1, min(splits, suffix_tiles)), 3.0 + step * -(-suffix_tiles // splits)
        for ours in sorted({-(-tiles // length) for length in range(1, tiles + 1)}):
            if ours > 32:
                break
            front_time = 3.0 + step * -(-tiles // ours)
            # the prefix's pieces start first; the suffixes fill the slots beside them, then those behind them
            rounds, front = divmod(units * ours - 1, slots)
            front += 1
            k = -(-back // slots)
            while (slots - front) * k + front * max(0, int((k * back_time - front_time) / back_time)) < back:
                k += 1
            time = max(rounds * front_time + max(front_time, k * back_time) + 3.0, least) + per_part * (ours + splits)
            found[tokens, ours, splits, ours + splits] = time
    return found


def _kernel_plans(n, rows, pieces, kv_heads, head_dim, tiles, expected, divisions, least, sms):
    """The prefix kernel beside the suffixes' launch. A CTA of it keeps an SM to itself while the others stream the suffixes,
    so the SMs are divided like the work: a prefix CTA takes about 14 us and 2 us more per step (128 keys for up to 256 rows;
    two tiles make a step when 128 rows are all there are, and it starts 3 us sooner), a suffix half an SM for 3.5 us and
    1.1 us per 128 keys (sequences of more than 16 rows: 1.5 us), or longer when all of them together are bound by memory;
    a part costs its fp32 rows, written and read once at 4 TB/s. With more
    prefix CTAs than 7 in 10 SMs the suffixes hardly run before they end (33 x 5 rows behind 4001 tokens: 28 us with 96 CTAs,
    37 us with 120)."""
    one_tile = rows <= _PREFIX_TILE
    units = kv_heads * (1 if one_tile else -(-rows // (2 * _PREFIX_TILE)))
    step = 1.1 if rows <= 16 * n else 1.5
    per_part = rows * kv_heads * head_dim * 8 / 4e6
    suffix_tiles = -(-expected // _PREFIX_TILE)
    found = {}
    for splits in divisions:
        if splits > max(1, 2 * sms // pieces) and splits > divisions[0]:
            break
        chain = 6.0 + 1.35 * -(-suffix_tiles // splits)
        many, each = pieces * splits, 3.5 + step * (expected / 256 + 0.5) / splits          # half of `expected` on average
        alone = max(many * each / (2 * sms), least - 3.0)          # all suffixes on all SMs
        for ours in range(1, min(tiles, 32) + 1):
            if ours > 1 and units * ours > sms:
                break
            parts = 2 * ours if one_tile and ours < tiles else ours
            if parts + splits > 64:
                continue
            last = 11.0 + -(-tiles // ours) if one_tile else 14.0 + 2.0 * -(-tiles // ours)
            done = min(1.0, last * 2 * max(0, sms - units * ours) / (many * each))          # of the suffixes, when the prefix ends
            time = max(least, chain, last + (1.0 - done) * alone) + 0.1 * last + (parts + splits) * per_part
            if 10 * units * ours > 7 * sms:
                time += 8.0 + alone
            found[0, ours, splits, parts + splits] = time
    return found


def shared_prefix_attention(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
                            context_lens: torch.Tensor, prefix_len: int, *, q_len: int = 1, scale: float | None = None,
                            max_context: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Paged attention of a batch of sequences that all begin with the same ``prefix_len`` cached tokens.

    Same result as :func:`paged_attention`, but the keys and values of the prefix are read once for the whole batch and
    multiplied with all its query rows at once. ``q`` is ``[n * q_len, Hq, hd]``, ``q_len`` newest tokens of every
    sequence one after another (1 for decoding, ``k + 1`` for verification, more for the chunk of a prompt); token
    ``j`` of sequence ``i`` attends to its first ``context_lens[i] - q_len + j + 1`` tokens. ``block_tables`` (int32
    ``[n, max_blocks]``) and ``context_lens`` (int32 ``[n]``, new tokens included) cover the whole context; the blocks
    of the prefix are taken from the first row. New tokens lie behind the prefix
    (``context_lens[i] - q_len >= prefix_len``): the whole prefix is visible to every row. A prefix that ends inside a
    block is shared up to that block. Heads are 64 or 128 wide, ``Hq / Hkv`` is at most 128.

    ``max_context``: a host-side bound on the context lengths from which the number of parts per sequence is chosen (without
    one: what the tables can hold, or 512 tokens behind the prefix if that is more than 1024). It bounds nothing that is
    read. A row whose sequence has no token at all, or whose visible scores are all minus infinity, comes out as zeros; NaN in a
    query or a visible key makes the row NaN, and what is not finite among the values of a sequence's tokens may reach all of its
    rows. ``scale`` (1e-30 to 1e3) defaults to ``1 / sqrt(hd)``; ``out``
    (contiguous, shaped like ``q``, 16-byte aligned, apart from the inputs) receives the result.
    """
    if out is None and native.fast is not None:
        found = native.fast.shared_prefix_attention(q, key_cache, value_cache, block_tables, context_lens, prefix_len, q_len, scale,
                                                    max_context, prefix_plan)
        if found is not None:
            native.launch_count += 2
            return found
    if q.dim() != 3 or key_cache.dim() != 4 or block_tables.dim() != 2:
        raise ValueError("shared_prefix_attention: q is [rows, heads, hd], the caches [blocks, block, kv_heads, hd], block_tables [n, max_blocks]")
    total, heads, head_dim = q.shape
    num_blocks, block_size, kv_heads, cache_dim = key_cache.shape
    n, max_blocks = block_tables.shape
    if q_len < 1 or total != n * q_len:
        raise ValueError(f"shared_prefix_attention: {total} query rows are not {q_len} for each of {n} sequences")
    if cache_dim != head_dim or kv_heads < 1 or heads < 1 or heads % kv_heads or num_blocks < 1 or max_blocks < 1:
        raise ValueError(f"shared_prefix_attention: {heads} query heads of {head_dim} do not go with {kv_heads} KV heads of {cache_dim}, "
                         "or the cache or the block tables are empty")
    if not 0 <= prefix_len <= max_blocks * block_size:
        raise ValueError(f"shared_prefix_attention: prefix_len {prefix_len} does not fit block tables of {max_blocks} blocks")
    index, dtype = q.get_device(), q.dtype
    if not (key_cache.dtype is value_cache.dtype is dtype and block_tables.dtype is context_lens.dtype is _I32
            and value_cache.shape == key_cache.shape and context_lens.shape == (n,)
            and key_cache.get_device() == index == value_cache.get_device() == block_tables.get_device() == context_lens.get_device()
            and key_cache.is_contiguous() and value_cache.is_contiguous() and block_tables.is_contiguous() and context_lens.is_contiguous()):
        for name, t, kind, shape in (("key_cache", key_cache, dtype, key_cache.shape), ("value_cache", value_cache, dtype, key_cache.shape),
                                     ("block_tables", block_tables, _I32, block_tables.shape), ("context_lens", context_lens, _I32, (n,))):
            _dense("shared_prefix_attention", name, t, kind, q.device, shape)
    if out is not None:
        _dense("shared_prefix_attention", "out", out, dtype, q.device, q.shape)
        if any(_overlap(out, t) for t in (q, key_cache, value_cache, block_tables, context_lens)):
            raise ValueError("shared_prefix_attention: out must not overlap the inputs")
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    elif not 1e-30 <= scale <= 1e3:
        # positive, as the reference maximum of a row is that of its unscaled scores, not zero in fp32, and not so large that the
        # rounding of scale * maximum (its 2^-24th) is an exponent of its own
        raise ValueError(f"shared_prefix_attention: scale must be positive, between 1e-30 and 1e3 (got {scale})")
    if index < 0:
        found = reference.shared_prefix_attention(q, key_cache, value_cache, block_tables, context_lens, prefix_len, q_len, scale)
        return found if out is None else out.copy_(found)
    if dtype is not _BF16:
        raise TypeError(f"shared_prefix_attention: CUDA tensors must be bfloat16 (got {dtype})")
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return shared_prefix_attention(q, key_cache, value_cache, block_tables, context_lens, prefix_len, q_len=q_len,
                                           scale=scale, max_context=max_context, out=out)
    q_at, pitch = q.data_ptr(), heads * head_dim
    if not q.is_contiguous():
        pitch = q.stride(0)
        if q.stride(2) != 1 or q.stride(1) != head_dim or pitch % 8:
            q, pitch = q.contiguous(), heads * head_dim
            q_at = q.data_ptr()
    if q_at % 16:
        q, pitch = q.clone(memory_format=_CONTIGUOUS), heads * head_dim
        q_at = q.data_ptr()
    if out is None:
        out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    if total == 0:
        return out
    shared = prefix_len // block_size * block_size
    group = heads // kv_heads
    room = max_blocks * block_size
    behind = room - shared
    if max_context is not None:          # in whole tiles: contexts that grow by a token per step keep their plan for 128 steps
        behind = -(-max(0, min(max_context, room) - shared) // _PREFIX_TILE) * _PREFIX_TILE
    prefix_tokens, prefix_splits, splits, parts = prefix_plan(n, q_len, group, kv_heads, head_dim, shared, behind, int(max_context is not None))
    # fp32 parts of every (row, head): un-normalised outputs, then (reference maximum, sum) pairs
    count = total * heads * parts
    workspace = torch.empty(count * (head_dim + 2), dtype=_F32, device=q.device)
    parts_at = workspace.data_ptr()
    native.call_packed("ajb_shared_prefix_attention", q_at, key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(),
                context_lens.data_ptr(), out.data_ptr(), pitch, n, num_blocks, block_size, max_blocks, heads, kv_heads,
                head_dim, q_len, shared, scale, prefix_tokens, prefix_splits, splits, parts, parts_at, parts_at + 4 * count * head_dim,
                native.stream_ptr(index))
    return out


# ----------------------------------------------------------------------------- logits processing


def process_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                   history_lens: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                   presence: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                   bias_ids: torch.Tensor | None = None, bias_values: torch.Tensor | None = None,
                   token_mask: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Penalties for repeated tokens, token biases and a grammar mask on ``logits`` ``[rows, vocab]`` (bf16 or fp32);
    returns new fp32 logits for the sampler. In this order, for token ``v`` of a row:

    * ``history`` (int32 ``[rows, width]``; the first ``prompt_lens[row]`` of its ``history_lens[row]`` tokens are the
      prompt, the rest was generated; ids outside the vocabulary are skipped): a logit of any token in it is divided
      by ``repetition[row]`` if positive, multiplied with it otherwise; then ``frequency[row]`` times the number of
      times ``v`` was generated is taken off, and ``presence[row]`` if it was generated at all (fp32 ``[rows]``,
      ``None`` = no such penalty);
    * ``bias_values[row, j]`` is added to token ``bias_ids[row, j]`` (fp32 / int32 ``[rows, biases]``, ids outside the
      vocabulary are skipped, equal ids are added one after another);
    * tokens whose bit is not set in ``token_mask`` (int32 ``[rows, ceil(vocab / 32)]``, bit ``v % 32`` of word
      ``v // 32``) become ``-inf``, whatever their logit was. A row whose mask leaves nothing is ``-inf`` throughout.

    ``out`` (fp32 ``[rows, vocab]``, contiguous, apart from the inputs) receives the result.
    """
    if out is None and native.fast is not None:
        found = native.fast.process_logits(logits, history, prompt_lens, history_lens, repetition, presence, frequency, bias_ids,
                                           bias_values, token_mask)
        if found is not None:
            native.launch_count += 1
            return found
    dtype, index = logits.dtype, logits.get_device()
    if dtype is not _BF16 and dtype is not _F32:
        raise TypeError(f"process_logits: logits must be bfloat16 or float32 (got {dtype})")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError("process_logits: logits must be [rows, vocab] with at least one token")
    rows, vocab = logits.shape
    each = (rows,)
    width = biases = 0
    if history is not None:
        if prompt_lens is None or history_lens is None or history.dim() != 2:
            raise ValueError("process_logits: history is [rows, width] and comes with prompt_lens and history_lens")
        width = history.shape[1]
        if not (history.dtype is prompt_lens.dtype is history_lens.dtype is _I32 and history.shape[0] == rows
                and prompt_lens.shape == each == history_lens.shape
                and history.get_device() == index == prompt_lens.get_device() == history_lens.get_device()
                and history.is_contiguous() and prompt_lens.is_contiguous() and history_lens.is_contiguous()):
            for name, t, shape in (("history", history, (rows, width)), ("prompt_lens", prompt_lens, each), ("history_lens", history_lens, each)):
                _dense("process_logits", name, t, _I32, logits.device, shape)
        for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
            if t is not None and not (t.dtype is _F32 and t.shape == each and t.get_device() == index and t.is_contiguous()):
                _dense("process_logits", name, t, _F32, logits.device, each)
    elif not (repetition is None and presence is None and frequency is None and prompt_lens is None and history_lens is None):
        raise ValueError("process_logits: penalties need a history")
    if bias_ids is not None or bias_values is not None:
        if bias_ids is None or bias_values is None or bias_ids.dim() != 2:
            raise ValueError("process_logits: bias_ids and bias_values come together, [rows, biases] each")
        biases = bias_ids.shape[1]
        if not (bias_ids.dtype is _I32 and bias_values.dtype is _F32 and bias_ids.shape == (rows, biases) == bias_values.shape
                and bias_ids.get_device() == index == bias_values.get_device() and bias_ids.is_contiguous() and bias_values.is_contiguous()):
            _dense("process_logits", "bias_ids", bias_ids, _I32, logits.device, (rows, biases))
            _dense("process_logits", "bias_values", bias_values, _F32, logits.device, (rows, biases))
    if token_mask is not None and not (token_mask.dtype is _I32 and token_mask.shape == (rows, (vocab + 31) // 32)
                                       and token_mask.get_device() == index and token_mask.is_contiguous()):
        _dense("process_logits", "token_mask", token_mask, _I32, logits.device, (rows, (vocab + 31) // 32))
    if out is not None:
        _dense("process_logits", "out", out, _F32, logits.device, (rows, vocab))
        if any(t is not None and _overlap(out, t) for t in (logits, history, prompt_lens, history_lens, repetition, presence, frequency,
                                                            bias_ids, bias_values, token_mask)):
            raise ValueError("process_logits: out must not overlap the inputs")
    if index < 0:
        found = reference.process_logits(logits, history, prompt_lens, history_lens, repetition, presence, frequency, bias_ids,
                                         bias_values, token_mask)
        return found if out is None else out.copy_(found)
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return process_logits(logits, history=history, prompt_lens=prompt_lens, history_lens=history_lens, repetition=repetition,
                                  presence=presence, frequency=frequency, bias_ids=bias_ids, bias_values=bias_values,
                                  token_mask=token_mask, out=out)
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    if out is None:
        out = torch.empty(rows, vocab, dtype=_F32, device=logits.device)
    native.call_packed("ajb_process_logits", logits.data_ptr(), 1 if dtype is _F32 else 0, logits.stride(0), out.data_ptr(),
                rows, vocab, _ptr(history) if width else 0, width, width, _ptr(prompt_lens), _ptr(history_lens),
                _ptr(repetition), _ptr(presence), _ptr(frequency), _ptr(bias_ids), _ptr(bias_values),
                biases, _ptr(token_mask), (vocab + 31) // 32, native.stream_ptr(index))
    return out
