"""Shared prefixes, logits processing and batch maps without a GPU: the operators' CPU forms against direct statements in
64 bits, their refusals, and the serving engine's use of them."""

import math
import random
from pathlib import Path

import pytest
import torch

from ajllm_b200.engine import LLMEngine, OutOfBlocks, PagedKVCache, SamplingParams
from ajllm_b200.engine.model_runner import ModelRunner, RunItem
from ajllm_b200.models import build_model
from ajllm_b200.ops import serving
from ajllm_b200.workflows.lm_generate import common_prefix

CFG = {"name": "p", "context_length": 160, "d_model": 64, "num_layers": 2, "num_heads": 4, "num_kv_heads": 2, "d_ff": 128,
       "init": {"type": "normal", "std": 0.2}}
VOCAB = 300
I32 = torch.int32


def _i32(values):
    return torch.tensor(values, dtype=I32)


# ----------------------------------------------------------------------------- operators

@pytest.mark.parametrize("block_size", [1, 4, 16])
def test_batch_maps_against_the_cache(block_size):
    cache = PagedKVCache(1, 200, block_size, 1, 8, torch.float32, torch.device("cpu"))
    pad = cache.allocator.allocate()
    rng = random.Random(block_size)
    cached = [0, 3, 17, 0, block_size, 9]
    new = [5, 1, 0, 0, 1, 20]
    slots, positions = [], []
    for i, (have, n) in enumerate(zip(cached, new)):
        cache.append_slots(i, have)
        slots += cache.append_slots(i, n)
        positions += range(have, have + n)
    blocks = [cache.tables[i].blocks for i in range(6)]
    ids = [b for own in blocks for b in own]
    width = max(map(len, blocks)) + rng.randint(0, 2)
    got = serving.batch_maps(_i32(ids), _i32([len(b) for b in blocks]), _i32(cached), _i32(new), sum(new) + 3, width,
                             block_size=block_size, pad_block=pad)
    assert got.tables.tolist() == [own + [pad] * (width - len(own)) for own in blocks]
    assert got.positions.tolist() == positions + [0] * 3
    assert got.slots.tolist() == slots + [pad * block_size] * 3 and got.slots.dtype is torch.int64
    assert got.q_start.tolist() == [0, 5, 6, 6, 6, 7, 27]
    assert got.context_lens.tolist() == [a + b for a, b in zip(cached, new)]
    buffers = serving.BatchMaps(*(torch.full_like(t, 7) for t in got))
    again = serving.batch_maps(_i32(ids), _i32([len(b) for b in blocks]), _i32(cached), _i32(new), sum(new) + 3, width,
                               block_size=block_size, pad_block=pad, out=buffers)
    assert all(a.data_ptr() == b.data_ptr() and torch.equal(a, c) for a, b, c in zip(again, buffers, got))


def test_batch_maps_without_sequences_and_with_missing_blocks():
    got = serving.batch_maps(_i32([]), _i32([]), _i32([]), _i32([]), 2, 3, pad_block=5)
    assert got.tables.shape == (0, 3) and got.q_start.tolist() == [0] and got.slots.tolist() == [80, 80]
    got = serving.batch_maps(_i32([4]), _i32([1]), _i32([15]), _i32([2]), 2, 1, pad_block=9)      # the second token has no block
    assert got.positions.tolist() == [15, 16] and got.slots.tolist() == [4 * 16 + 15, 9 * 16]


def test_batch_maps_of_lengths_past_32_bits():
    """As on a GPU: positions and context lengths stop at the largest int32, tokens without a block go to the pad block."""
    big = 2**31 - 1
    got = serving.batch_maps(_i32([5, 6]), _i32([1, 1]), _i32([big - 1, big]), _i32([3, big]), 5, 1, pad_block=9)
    assert got.positions.tolist() == [big - 1] + [big] * 4 and got.context_lens.tolist() == [big, big]
    assert got.slots.tolist() == [9 * 16 + (big - 1 + j) % 16 for j in (0, 1, 2, 1, 2)] and got.q_start.tolist() == [0, 3, 5]


@pytest.mark.parametrize("change", [
    {"total_tokens": -1}, {"max_blocks": 0}, {"block_size": 0}, {"pad_block": -1},
    {"block_ids": torch.zeros(2, dtype=torch.int64)}, {"block_ids": torch.zeros(1, 2, dtype=I32)},
    {"block_counts": torch.zeros(2, dtype=I32)}, {"cached_lens": torch.zeros(1)}, {"q_lens": torch.zeros(4, dtype=I32)[::2][:1].expand(2)},
    {"block_ids": torch.zeros(4, dtype=I32)[::2]}])
def test_batch_maps_refuses(change):
    call = dict(block_ids=_i32([0, 1]), block_counts=_i32([2]), cached_lens=_i32([3]), q_lens=_i32([1]), total_tokens=1, max_blocks=2)
    serving.batch_maps(**call)
    with pytest.raises((ValueError, TypeError)):
        serving.batch_maps(**{**call, **change})


def test_batch_maps_refuses_outputs_of_another_shape():
    call = (_i32([0, 1]), _i32([2]), _i32([3]), _i32([1]), 1, 2)
    good = serving.batch_maps(*call)
    for i in range(5):
        out = list(good)
        out[i] = torch.zeros(good[i].numel() + 1, dtype=good[i].dtype)
        with pytest.raises((ValueError, TypeError)):
            serving.batch_maps(*call, out=tuple(out))


def test_batch_maps_refuses_outputs_over_its_inputs():
    ids, counts, cached, new = _i32([0, 1]), _i32([2]), _i32([3]), _i32([1])
    good = serving.batch_maps(ids, counts, cached, new, 1, 2)
    for out in (good._replace(context_lens=cached), good._replace(q_start=good.tables.flatten())):
        with pytest.raises(ValueError, match="apart"):
            serving.batch_maps(ids, counts, cached, new, 1, 2, out=out)


def _paged(contexts, shared, kv_heads=2, hd=8, block_size=4):
    """A cache of sequences that share their first ``shared`` tokens, its block tables, and each sequence's own keys and values."""
    gen = torch.Generator().manual_seed(len(contexts) + shared)
    cache = PagedKVCache(1, 64, block_size, kv_heads, hd, torch.float32, torch.device("cpu"))
    whole = shared // block_size * block_size
    cache.allocator.allocate()
    cache.append_slots(99, whole)
    cache.keys.normal_(generator=gen)
    cache.values.normal_(generator=gen)
    for i, context in enumerate(contexts):
        cache.fork(99, i)
        cache.append_slots(i, context - whole)
    return cache, cache.block_table_tensor(list(range(len(contexts))), torch.device("cpu"))


@pytest.mark.parametrize("contexts,shared,q_len", [([5, 9, 30], 4, 1), ([12, 13, 9], 8, 1), ([11, 20], 7, 3), ([6, 3, 9], 0, 2), ([10], 9, 1)])
def test_shared_prefix_attention_against_64_bits(contexts, shared, q_len):
    cache, tables = _paged(contexts, shared)
    heads, hd = 4, 8
    q = torch.randn(len(contexts) * q_len, heads, hd, generator=torch.Generator().manual_seed(1))
    got = serving.shared_prefix_attention(q, cache.keys[0], cache.values[0], tables, _i32(contexts), shared, q_len=q_len)
    for i, context in enumerate(contexts):
        keys, values = (c[0][tables[i].long()].reshape(-1, 2, hd).double().repeat_interleave(2, dim=1) for c in (cache.keys, cache.values))
        for j in range(q_len):
            seen = context - q_len + j + 1
            scores = torch.einsum("hd,shd->hs", q[i * q_len + j].double(), keys[:seen]) / math.sqrt(hd)
            want = torch.einsum("hs,shd->hd", scores.softmax(-1), values[:seen])
            # fp32 dot products of 8, a softmax and a sum over at most 30 keys: some 50 roundings of 2^-24
            assert float((got[i * q_len + j].double() - want).abs().max()) < 50 * 2 ** -24 * float(values.abs().max())


def test_only_rows_without_a_key_are_zero():
    """A row that sees nothing is zeros; one whose query or visible key holds a NaN is not, with and without a prefix."""
    for contexts, shared in (([6, 0, 9], 0), ([9, 12, 10], 8)):
        cache, tables = _paged([max(1, c) for c in contexts], shared)
        q = torch.randn(3, 4, 8, generator=torch.Generator().manual_seed(2))
        q[0, 1, 0] = math.nan
        got = serving.shared_prefix_attention(q, cache.keys[0], cache.values[0], tables, _i32(contexts), shared)
        rows = got.isnan().all(-1)
        assert rows[0].tolist() == [False, True, False, False] and int(got.isnan().any(-1).sum()) == 1
        assert (torch.count_nonzero(got[1]) == 0) == (contexts[1] == 0)
        cache.keys[0][tables[2, 0], 1, 0, 3] = math.nan                 # KV head 0: query heads 0 and 1
        got = serving.shared_prefix_attention(q, cache.keys[0], cache.values[0], tables, _i32(contexts), shared)
        assert got.isnan().all(-1)[2].tolist() == [True, True, False, False]


@pytest.mark.parametrize("contexts,shared", [([6, 4, 9], 0), ([9, 12, 10], 8)])
def test_rows_of_scores_that_are_all_minus_infinity_are_zero(contexts, shared):
    cache, tables = _paged(contexts, shared)
    q = torch.randn(3, 4, 8, generator=torch.Generator().manual_seed(2))
    cache.keys[0].abs_()
    q[1, 2], q[2, 3] = -math.inf, -1e30
    got = serving.shared_prefix_attention(q, cache.keys[0], cache.values[0], tables, _i32(contexts), shared)
    assert torch.count_nonzero(got[1, 2]) == 0 and torch.isfinite(got).all() and torch.count_nonzero(got) == 11 * 8


def _attention_call():
    cache, tables = _paged([9, 12], 8)
    return dict(q=torch.zeros(2, 4, 8), key_cache=cache.keys[0], value_cache=cache.values[0], block_tables=tables,
                context_lens=_i32([9, 12]), prefix_len=8)


@pytest.mark.parametrize("change", [
    {"q": torch.zeros(3, 4, 8)}, {"q": torch.zeros(2, 3, 8)}, {"q": torch.zeros(2, 4, 16)}, {"q": torch.zeros(8, 8)}, {"q_len": 0}, {"q_len": 2},
    {"prefix_len": -1}, {"prefix_len": 13}, {"context_lens": torch.zeros(2, dtype=torch.int64)}, {"context_lens": torch.zeros(3, dtype=I32)},
    {"block_tables": torch.zeros(2, 3)}, {"block_tables": torch.zeros(3, 3, dtype=I32)}, {"block_tables": torch.zeros(2, 6, dtype=I32)[:, ::2]},
    {"value_cache": torch.zeros(64, 4, 2, 4)}, {"key_cache": torch.zeros(64, 4, 2, 8).double()}, {"out": torch.zeros(2, 4, 9)},
    {"out": torch.zeros(2, 4, 8).double()}, {"out": torch.zeros(2, 4, 16)[..., ::2]},
    {"scale": 0.0}, {"scale": -0.1}, {"scale": math.nan}, {"scale": math.inf}])
def test_shared_prefix_attention_refuses(change):
    call = _attention_call()
    serving.shared_prefix_attention(**call)
    with pytest.raises((ValueError, TypeError)):
        serving.shared_prefix_attention(**{**call, **change})


@pytest.mark.parametrize("scale", [1e-46, 1e-40, 9e-31, 1.1e3, 1e39, 1e300])
def test_shared_prefix_attention_refuses_a_scale_that_fp32_arithmetic_loses(scale):
    call = _attention_call()
    with pytest.raises(ValueError, match="between"):
        serving.shared_prefix_attention(**call, scale=scale)
    for kept in (1e-30, 1e3, 1):
        assert torch.isfinite(serving.shared_prefix_attention(**call, scale=kept)).all()


def test_shared_prefix_attention_refuses_its_query_as_output():
    call = _attention_call()
    with pytest.raises(ValueError, match="overlap"):
        serving.shared_prefix_attention(**call, out=call["q"])


def test_division_of_shared_prefix_attention_is_one_that_the_kernels_take(monkeypatch):
    """Over the whole range of sizes: the limits that the entry point checks, and every key in some part."""
    monkeypatch.setattr(serving, "_SM_COUNT", [148])
    rng = random.Random(4)
    for _ in range(4000):
        n, q_len = int(2 ** rng.uniform(0, 10)), rng.choice([1, 1, 1, 2, 5, 17, 300])
        group, kv_heads, hd = rng.choice([1, 2, 4, 6, 8, 16, 32, 71, 128]), rng.choice([1, 2, 8, 16, 32]), rng.choice([64, 128])
        shared, behind = 16 * int(2 ** rng.uniform(-1, 11)), int(2 ** rng.uniform(-1, 15))
        tokens, ours, splits, parts = serving.prefix_plan(n, q_len, group, kv_heads, hd, shared, behind, rng.choice([0, 1]))
        tiles, rows = -(-shared // 128), n * q_len * group
        if not shared:
            assert (tokens, ours) == (0, 0) and parts == splits >= 1
            continue
        assert 1 <= ours <= min(tiles, 32) and 1 <= splits <= 16 and parts <= 64
        assert tokens == 0 or (tokens * group <= 32 and q_len * group <= 32)
        twice = tokens == 0 and rows <= 128 and ours < tiles
        assert parts == splits + (2 * ours if twice else ours)


def test_parts_of_paged_attention_where_pairs_nearly_fill_the_device(monkeypatch):
    """Long contexts are left whole only where that is the faster form: up to 32 rows of 128-wide heads."""
    monkeypatch.setattr(serving, "_SM_COUNT", [148])
    for pairs in (120, 128, 148):
        assert serving.paged_splits(pairs, 4096) == serving.paged_splits(pairs, 4096, 32, 128) == 1
        for rows, hd in ((33, 128), (64, 128), (40, 64), (8, 64)):
            assert serving.paged_splits(pairs, 4096, rows, hd) == 2 and serving.paged_splits(pairs, 1000, rows, hd) == 1
    assert serving.paged_splits(149, 1 << 17, 40, 64) == serving.paged_splits(149, 1 << 17) == 1


def _formula(x, history, prompt, total, repetition, presence, frequency, biases, allowed):
    """One row of processed logits, token by token, in 64 bits."""
    out = []
    known = [t for t in history[:total] if 0 <= t < len(x)]
    made = [t for t in history[prompt:total] if 0 <= t < len(x)]
    for v, value in enumerate(x):
        if v in known:
            value = value / repetition if value > 0 else value * repetition
        count = made.count(v)
        if count:
            value = value - frequency * count - presence
        value += sum(b for t, b in biases if t == v)
        out.append(value if allowed is None or v in allowed else -math.inf)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 31, 32, 77])
def test_process_logits_against_the_formula(vocab, dtype):
    rng = random.Random(vocab)
    rows, width = 5, 12
    logits = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(vocab)).to(dtype)
    history = [[rng.randint(-2, vocab + 2) for _ in range(width)] for _ in range(rows)]
    prompt, total = [0, 3, 12, 5, 7], [0, 12, 12, 5, 9]
    repetition, presence, frequency = [1.0, 1.3, 0.8, 2.0, 1.1], [0.0, 0.5, 0.1, -0.3, 1.0], [0.0, 0.25, 0.5, 0.0, -0.125]
    biases = [[(rng.randint(-1, vocab), rng.uniform(-3, 3)) for _ in range(4)] for _ in range(rows)]
    allowed = [{v for v in range(vocab) if rng.random() < 0.5} for _ in range(rows - 1)] + [set()]
    words = (vocab + 31) // 32
    mask = torch.zeros(rows, words, dtype=I32)
    for row, tokens in enumerate(allowed):
        for v in tokens:
            mask[row, v // 32] |= torch.tensor((1 << (v % 32)) - ((v % 32 == 31) << 32), dtype=I32)
    f32 = lambda values: torch.tensor(values, dtype=torch.float32)
    got = serving.process_logits(logits, history=_i32(history), prompt_lens=_i32(prompt), history_lens=_i32(total), repetition=f32(repetition),
                                 presence=f32(presence), frequency=f32(frequency), bias_ids=_i32([[t for t, _ in b] for b in biases]),
                                 bias_values=f32([[v for _, v in b] for b in biases]), token_mask=mask)
    assert got.dtype is torch.float32
    for row in range(rows):
        want = torch.tensor(_formula(logits[row].double().tolist(), history[row], prompt[row], total[row], repetition[row], presence[row],
                                     frequency[row], biases[row], allowed[row]), dtype=torch.float64)
        assert torch.equal(torch.isinf(got[row]), torch.isinf(want))
        kept = ~torch.isinf(want)
        # at most eight fp32 operations on values below 20, and parameters rounded to fp32
        assert not kept.any() or float((got[row].double() - want)[kept].abs().max()) < 16 * 2 ** -24 * 20


def test_process_logits_masks_whatever_the_logit_was():
    logits = torch.tensor([[math.inf, math.nan, -math.inf, 1.0, torch.finfo(torch.float32).min]])
    got = serving.process_logits(logits, token_mask=_i32([[0b11000]]))
    assert got.tolist() == [[-math.inf] * 3 + [1.0, torch.finfo(torch.float32).min]]
    assert serving.process_logits(logits[:0], token_mask=torch.zeros(0, 1, dtype=I32)).shape == (0, 5)


@pytest.mark.parametrize("change", [
    {"logits": torch.zeros(2, 40).half()}, {"logits": torch.zeros(40)}, {"logits": torch.zeros(2, 0)}, {"logits": torch.zeros(3, 40)},
    {"history": None}, {"prompt_lens": None}, {"history": torch.zeros(2, 5)}, {"history": torch.zeros(2, 10, dtype=I32)[:, ::2]},
    {"history_lens": torch.zeros(1, dtype=I32)}, {"repetition": torch.ones(2).double()}, {"presence": torch.ones(3)}, {"frequency": torch.ones(2, 1)},
    {"bias_ids": None}, {"bias_values": None}, {"bias_values": torch.zeros(2, 4)}, {"bias_ids": torch.zeros(2, 3)},
    {"token_mask": torch.zeros(2, 1, dtype=I32)}, {"token_mask": torch.zeros(2, 2)}, {"out": torch.zeros(2, 40).bfloat16()}, {"out": torch.zeros(2, 41)}])
def test_process_logits_refuses(change):
    call = dict(logits=torch.zeros(2, 40), history=torch.zeros(2, 5, dtype=I32), prompt_lens=_i32([1, 2]), history_lens=_i32([3, 4]),
                repetition=torch.ones(2), presence=torch.ones(2), frequency=torch.ones(2), bias_ids=torch.zeros(2, 3, dtype=I32),
                bias_values=torch.zeros(2, 3), token_mask=torch.zeros(2, 2, dtype=I32))
    serving.process_logits(**call)
    with pytest.raises((ValueError, TypeError)):
        serving.process_logits(**{**call, **change})


def test_process_logits_refuses_its_input_as_output():
    logits = torch.zeros(2, 40)
    with pytest.raises(ValueError, match="overlap"):
        serving.process_logits(logits, out=logits)


# ----------------------------------------------------------------------------- cache

def test_forked_sequences_know_what_they_share():
    cache = PagedKVCache(1, 16, 4, 1, 8, torch.float32, torch.device("cpu"))
    cache.append_slots(-1, 8)
    cache.fork(-1, 0)
    cache.append_slots(0, 5)
    assert cache.shares(0, -1, 2) and not cache.shares(0, -2, 2) and not cache.shares(0, -1, 3) and not cache.shares(5, -1, 0)
    cache.truncate(0, 8)
    assert cache.shares(0, -1, 2)
    cache.truncate(0, 4)
    assert not cache.shares(0, -1, 2) and cache.shares(0, -1, 1)
    cache.append_slots(0, 8)
    assert not cache.shares(0, -1, 2)          # the second block is another one now
    cache.free(0)
    cache.free(-1)
    assert cache.allocator.free_blocks == 16


# ----------------------------------------------------------------------------- engine

@pytest.fixture(scope="module")
def model():
    torch.manual_seed(0)
    return build_model(CFG, VOCAB)


def _prompts(prefix=37, tails=(1, 5, 20, 3, 9)):
    gen = torch.Generator().manual_seed(8)
    head = torch.randint(0, VOCAB, (prefix,), generator=gen).tolist()
    return head, [head + torch.randint(0, VOCAB, (n,), generator=gen).tolist() for n in tails]


def _count_calls(monkeypatch, name):
    calls = []
    real = getattr(serving, name)
    monkeypatch.setattr(serving, name, lambda *a, **k: calls.append(k) or real(*a, **k))
    return calls


def test_engine_with_a_shared_prefix_generates_the_same(model, monkeypatch):
    head, prompts = _prompts()
    prompts.append([7, 8, 9])                                   # does not begin with it
    params = SamplingParams(10, 0.0, None)
    want = [o.output for o in LLMEngine(model, block_size=8, num_blocks=200).generate(prompts, params)]
    calls = _count_calls(monkeypatch, "shared_prefix_attention")
    engine = LLMEngine(model, block_size=8, num_blocks=200)
    assert engine.share_prefix(head) == 32
    assert [o.output for o in engine.generate(prompts, params)] == want
    assert not calls                                            # one request does not share it: each reads its own context
    assert [o.output for o in engine.generate(prompts[:5], params)] == want[:5]
    assert len(calls) == CFG["num_layers"] * 9                  # every step but the ragged prefill
    assert engine.stats.prompt_tokens == 2 * sum(len(p) - 32 for p in prompts[:5]) + 3
    assert engine.cache.allocator.free_blocks == 200 - 4
    engine.release_prefix()
    engine.release_prefix()
    assert engine.cache.allocator.free_blocks == 200
    assert [o.output for o in engine.generate(prompts, params)] == want


def test_prompts_inside_the_prefix_and_one_token_behind_it(model):
    head, prompts = _prompts(prefix=32, tails=(0, 1, 1, 2))
    prompts.append(head[:20])
    params = SamplingParams(6, 0.0, None)
    want = [o.output for o in LLMEngine(model, block_size=8, num_blocks=200).generate(prompts, params)]
    engine = LLMEngine(model, block_size=8, num_blocks=200)
    assert engine.share_prefix(head) == 32
    assert [o.output for o in engine.generate(prompts, params)] == want


def test_shared_prefix_survives_preemption_release_and_another_prefix(model):
    head, prompts = _prompts()
    params = SamplingParams(12, 0.0, None)
    want = [o.output for o in LLMEngine(model, block_size=8, num_blocks=200).generate(prompts, params)]
    engine = LLMEngine(model, block_size=8, num_blocks=14)      # 4 blocks of prefix, 5 of the longest tail
    assert engine.share_prefix(head) == 32
    assert [o.output for o in engine.generate(prompts, params)] == want
    assert engine.stats.preemptions > 0 and engine.cache.allocator.free_blocks == 10
    ids = [engine.add_request(p, params) for p in prompts]
    found = {o.request_id: o for _ in range(3) for o in engine.step()}
    engine.release_prefix()                                     # its blocks are still in use
    assert engine.share_prefix(prompts[0][:9]) == 8
    while engine.has_unfinished():
        found.update((o.request_id, o) for o in engine.step())
    assert [found[i].output for i in ids] == want
    engine.release_prefix()
    assert engine.cache.allocator.free_blocks == 14


def test_share_prefix_refuses(model):
    engine = LLMEngine(model, block_size=8, num_blocks=24)
    assert engine.share_prefix([1, 2, 3]) == 0 and engine.scheduler.prefix is None
    with pytest.raises(ValueError, match="vocabulary"):
        engine.share_prefix([VOCAB] * 20)
    small = LLMEngine(model, block_size=8, num_blocks=2)
    with pytest.raises(OutOfBlocks):
        small.share_prefix([1] * 40)
    assert small.cache.allocator.free_blocks == 2
    assert engine.share_prefix([1] * 1000) == 152               # a token is left for every request
    with pytest.raises(ValueError, match="release"):
        engine.share_prefix([1] * 20)
    engine.add_request([2] * 60)
    with pytest.raises(RuntimeError, match="release"):
        engine.step()
    with pytest.raises(ValueError, match="draft"):
        LLMEngine(model, num_blocks=50, draft_model=model).share_prefix([1] * 40)


def test_share_prefix_frees_its_blocks_when_the_model_fails(model, monkeypatch):
    engine = LLMEngine(model, block_size=8, num_blocks=24)
    monkeypatch.setattr(engine.runner, "forward", lambda items: engine.cache.append_slots(items[0].seq_id, 8) and 1 / 0)
    with pytest.raises(ZeroDivisionError):
        engine.share_prefix([1] * 40)
    assert engine.cache.allocator.free_blocks == 24 and engine.scheduler.prefix is None


def test_prefix_longer_than_a_step(model):
    head, prompts = _prompts(prefix=64)
    params = SamplingParams(5, 0.0, None)
    want = [o.output for o in LLMEngine(model, block_size=8, num_blocks=200).generate(prompts, params)]
    engine = LLMEngine(model, block_size=8, num_blocks=200, max_batched_tokens=10)
    assert engine.share_prefix(head) == 64
    assert [o.output for o in engine.generate(prompts, params)] == want


def test_runner_steps_of_equal_chunks_behind_a_prefix(model):
    """Equal chunks of several tokens behind the prefix go through the shared form too, ragged ones do not."""
    head, prompts = _prompts(prefix=32, tails=(3, 3))
    logits = []
    for shared in (False, True):
        cache = PagedKVCache(2, 40, 8, 2, 16, torch.float32, torch.device("cpu"))
        runner = ModelRunner(model, cache)
        runner.forward([RunItem(-1, head, 0)])
        for i in range(2):
            cache.fork(-1, i)
        if shared:
            runner.set_prefix((-1, 32))
        items = [RunItem(i, p[32:], 3) for i, p in enumerate(prompts)]
        assert runner._shared_tokens(items) == (32 if shared else 0)
        assert runner._shared_tokens(items[:1]) == 0 and runner._shared_tokens([items[0], RunItem(1, [1], 1)]) == 0
        logits.append(runner.forward(items))
    assert float((logits[0] - logits[1]).abs().max()) < 1e-4 * float(logits[0].abs().max())


def test_common_prefix():
    assert common_prefix([]) == []
    assert common_prefix([[1, 2, 3], [1, 2, 4], [1, 2]]) == [1]
    assert common_prefix([[1, 2, 3]] * 2) == [1, 2]
    assert common_prefix([[1, 2], [2, 2]]) == []


# ----------------------------------------------------------------------------- engine: logits processing

def _words(allowed):
    words = torch.zeros((VOCAB + 31) // 32, dtype=torch.int64)
    for v in allowed:
        words[v // 32] |= 1 << (v % 32)
    return (words - ((words >> 31) << 32)).to(I32)


def test_engine_applies_penalties_like_the_formula(model):
    """Greedy decoding with penalties, request by request, against the formula on the model's own logits."""
    _, prompts = _prompts()
    params = [SamplingParams(12, 0.0, None, repetition_penalty=1.5), SamplingParams(12, 0.0, None, presence_penalty=2.0, frequency_penalty=1.0),
              SamplingParams(12, 0.0, None), SamplingParams(9, 0.0, None, logit_bias={5: 40.0, 9: 39.5}, frequency_penalty=0.25),
              SamplingParams(12, 0.0, None, frequency_penalty=-3.0)]
    outs = LLMEngine(model, block_size=8, num_blocks=30, max_num_seqs=3).generate(prompts, params)
    for prompt, p, out in zip(prompts, params, outs):
        assert len(out.output) == p.max_new_tokens
        tokens = list(prompt)
        for token in out.output:
            with torch.no_grad():
                x = model(torch.tensor([tokens]))[0, -1].double().tolist()
            want = _formula(x, tokens, len(prompt), len(tokens), p.repetition_penalty, p.presence_penalty, p.frequency_penalty,
                            list((p.logit_bias or {}).items()), None)
            assert want[token] > max(want) - 1e-3
            tokens.append(token)
    assert set(outs[3].output) == {5, 9}


def test_engine_without_processing_does_not_call_it(model, monkeypatch):
    calls = _count_calls(monkeypatch, "process_logits")
    LLMEngine(model, block_size=8, num_blocks=60).generate(_prompts()[1], SamplingParams(3, 0.7, 0.9))
    assert not calls


def test_engine_follows_a_token_mask_to_its_end(model):
    """A grammar of three tokens: what may follow depends on the output, and in the end nothing may."""
    steps = [{10, 11}, {200, 299}, {31, 32}]
    seen = []

    def grammar(output):
        seen.append(list(output))
        return _words(steps[len(output)] if len(output) < 3 else set())

    _, prompts = _prompts()
    params = [SamplingParams(8, 0.0, None, token_mask=grammar), SamplingParams(8, 1.0, 0.9),
              SamplingParams(8, 0.8, 0.95, token_mask=lambda output: None),
              SamplingParams(8, 1.0, None, token_mask=lambda output: _words({7}))]
    engine = LLMEngine(model, block_size=8, num_blocks=60)
    outs = engine.generate(prompts[:4], params)
    assert outs[0].finish_reason == "mask" and len(outs[0].output) == 3
    assert all(token in allowed for token, allowed in zip(outs[0].output, steps))
    assert [len(s) for s in seen] == [0, 1, 2, 3]
    assert [o.finish_reason for o in outs[1:]] == ["length"] * 3 and outs[3].output == [7] * 8
    assert engine.cache.allocator.free_blocks == 60
    # a request's draws do not depend on what the requests beside it are masked to
    alone = LLMEngine(model, block_size=8, num_blocks=60).generate([prompts[0], prompts[1]], [SamplingParams(1, 0.0, None), params[1]])
    assert alone[1].output == outs[1].output


def test_processing_holds_nothing_for_finished_requests(model):
    engine = LLMEngine(model, block_size=8, num_blocks=60, max_num_seqs=2)
    for _ in range(3):
        engine.generate(_prompts()[1], SamplingParams(4, 0.0, None, presence_penalty=1.0))
    assert not engine._processor._slots and not engine._processor._filled
    assert sorted(engine._processor._free) == list(range(len(engine._processor._free))) and len(engine._processor._free) <= 2


@pytest.mark.parametrize("change", [{"repetition_penalty": 0.0}, {"repetition_penalty": -1.0}, {"repetition_penalty": math.nan},
                                    {"presence_penalty": math.inf}, {"frequency_penalty": math.nan}, {"logit_bias": {VOCAB: 1.0}},
                                    {"logit_bias": {-1: 1.0}}, {"logit_bias": {3: math.nan}}, {"logit_bias": {3: -math.inf}}, {"token_mask": 5}])
def test_engine_refuses_parameters(model, change):
    engine = LLMEngine(model, block_size=8, num_blocks=30)
    with pytest.raises(ValueError):
        engine.add_request([1], SamplingParams(4, 0.0, None, **change))
    assert not engine.has_unfinished()


def test_engine_refuses_processing_with_a_draft_model_and_masks_of_another_shape(model):
    with pytest.raises(ValueError, match="draft"):
        LLMEngine(model, num_blocks=50, draft_model=model).add_request([1], SamplingParams(4, presence_penalty=1.0))
    for wrong in (torch.zeros(3, dtype=I32), torch.ones(VOCAB, dtype=torch.bool)):
        engine = LLMEngine(model, num_blocks=50)
        engine.add_request([1], SamplingParams(4, token_mask=lambda output: wrong))
        with pytest.raises(ValueError, match="token_mask"):
            engine.step()


def test_a_mask_that_raises_leaves_the_request_as_it_was(model):
    _, prompts = _prompts()
    want = LLMEngine(model, num_blocks=60).generate(prompts[:2], SamplingParams(6, 0.0, None))
    broken = [False]

    def mask(output):
        if broken[0]:
            raise KeyError("no such state")
        return None

    engine = LLMEngine(model, num_blocks=60)
    ids = [engine.add_request(prompts[0], SamplingParams(6, 0.0, None, token_mask=mask)), engine.add_request(prompts[1], SamplingParams(6, 0.0, None))]
    found = {}
    for step in range(20):
        broken[0] = step in (0, 2, 3)
        if broken[0]:
            with pytest.raises(KeyError):
                engine.step()
        else:
            found.update((o.request_id, o.output) for o in engine.step())
    assert [found[i] for i in ids] == [o.output for o in want]


def test_everything_together(model):
    """Shared prefix, batch of different penalties and a grammar: the same as one request at a time without sharing."""
    head, prompts = _prompts()
    params = [SamplingParams(9, 0.0, None, repetition_penalty=1.2), SamplingParams(9, 0.0, None),
              SamplingParams(9, 0.0, None, token_mask=lambda output: _words(range(len(output), VOCAB, 7))),
              SamplingParams(9, 0.0, None, logit_bias={4: 1.0, 8: -2.0}), SamplingParams(9, 0.0, None, frequency_penalty=0.7)]
    want = [LLMEngine(model, block_size=8, num_blocks=60).generate([prompt], p)[0].output for prompt, p in zip(prompts, params)]
    engine = LLMEngine(model, block_size=8, num_blocks=60)
    engine.share_prefix(head)
    assert [o.output for o in engine.generate(prompts, params)] == want


def test_lm_generate_shares_the_prompts_beginning_and_penalises(tmp_path):
    from ajllm_b200.workflows import lm_generate, lm_train
    from tests.helpers import loaded, make_project, prepare_artifacts, train_config
    project = make_project(tmp_path)
    prepare_artifacts(project)
    run = lm_train.run(loaded(project, train_config(project, max_steps=1)))["run_directory"]
    config = {"name": "g", "run_directory": run, "checkpoint": "final", "prompts": ["The night train", "The night train ran", "The night"],
              "max_new_tokens": 8, "temperature": 0.0, "samples_per_prompt": 2, "device": "cpu"}

    def texts(**changes):
        out = lm_generate.run(loaded(project, {**config, **changes}))
        return [c["text"] for r in out["results"] for c in r["completions"]], out["parameters"]

    plain, parameters = texts()
    assert texts(engine={"share_prefix": True, "block_size": 1})[0] == plain and "logit_bias" not in parameters
    biased, parameters = texts(logit_bias={65: 1000.0}, frequency_penalty=0.5)
    assert [text.rstrip("A") for text in biased] == [p for p in config["prompts"] for _ in range(2)]
    assert all(text.endswith("A" * 6) for text in biased)          # 8 where the context has room for them
    assert parameters["logit_bias"] == {65: 1000.0} and parameters["frequency_penalty"] == 0.5


def test_lm_generate_shares_the_beginning_of_what_is_left_of_prompts_that_are_too_long(tmp_path):
    """Prompts past the context length lose their beginning: what they share behind it is shared, not what was cut off."""
    from ajllm_b200.workflows import lm_generate, lm_train
    from tests.helpers import loaded, make_project, prepare_artifacts, train_config
    project = make_project(tmp_path)
    prepare_artifacts(project)
    run = lm_train.run(loaded(project, train_config(project, max_steps=1)))["run_directory"]
    config = {"name": "g", "run_directory": run, "checkpoint": "final", "prompts": ["The night train ran " * 40 + end for end in ("a", "b", "c")],
              "max_new_tokens": 3, "temperature": 0.0, "device": "cpu"}

    def texts(**engine):
        out = lm_generate.run(loaded(project, {**config, "engine": {"block_size": 1, "max_num_seqs": 1, **engine}}))
        return [c["text"] for r in out["results"] for c in r["completions"]]

    assert texts(share_prefix=True) == texts()


def test_the_extension_leaves_cpu_tensors_alone():
    """With the kernel library loaded, CPU calls still take the plain statements, and wrong ones their own errors."""
    from ajllm_b200.ops import native
    if not native.available():
        pytest.skip("the kernel library is not built")
    assert native.fast is not None
    maps = (_i32([3, 4]), _i32([1, 1]), _i32([2, 0]), _i32([1, 1]))
    assert native.fast.batch_maps(*maps, 2, 2, 16, 0, None) is None and native.fast.batch_maps() is None
    assert serving.batch_maps(*maps, 2, 2).slots.tolist() == [3 * 16 + 2, 4 * 16]
    assert native.fast.process_logits(*[None] * 10) is None and native.fast.process_logits(torch.zeros(1, 2), *[None] * 9) is None
    assert serving.process_logits(torch.ones(1, 2)).tolist() == [[1.0, 1.0]]
    call = _attention_call()
    serving.shared_prefix_attention(**call)
    assert native.fast.shared_prefix_attention(*call.values(), 1, None, None, serving.prefix_plan) is None
    for wrong in (dict(prefix_len="8"), dict(q=None), dict(block_tables=3)):
        with pytest.raises((TypeError, AttributeError, ValueError)):
            serving.shared_prefix_attention(**{**call, **wrong})


def test_launches_that_start_early_do_not_read_through_the_read_only_path():
    """A kernel that runs before its inputs are written (up to its wait for them) must not promise the compiler and the caches
    that they do not change."""
    sources = Path(serving.__file__).resolve().parent.parent / "csrc"
    early = [path for path in sources.glob("*.cu") if "griddepcontrol.wait" in path.read_text()]
    assert {path.stem for path in early} >= {"batch_maps", "logits", "paged_attention", "prefix_attention"}
    for path in early:
        for promise in ("__ldg", "ld_nc", "__restrict__", "ld.global.nc"):
            assert promise not in path.read_text(), (path.name, promise)
