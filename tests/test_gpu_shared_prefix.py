"""Block tables and slot maps, shared-prefix attention and logits processing on a GPU, against plain statements in
64 bits, at the sizes and masks where they can go wrong."""

import math
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from ajllm_b200.ops import native, reference, serving

pytestmark = pytest.mark.gpu

HALF_BF16 = 2.0 ** -8           # half a step of bf16, relative
HALF_FP32 = 2.0 ** -24


def _dev():
    return torch.device("cuda", 0)


def _i32(values, device=None):
    return torch.tensor(values, dtype=torch.int32, device=device or _dev())


# --------------------------------------------------------------------------------------------- batch maps


MAPS = [
    # block ids, counts, cached, new, total, max_blocks, block, pad
    (dict(counts=[1], cached=[0], new=[1]), 1, 1, 16),
    (dict(counts=[3, 1, 2], cached=[17, 0, 31], new=[31, 16, 1]), 48, 3, 16),
    (dict(counts=[2, 0, 0, 5], cached=[0, 0, 0, 70], new=[0, 0, 0, 7]), 7, 7, 16),            # sequences without tokens
    (dict(counts=[2, 4], cached=[30, 5], new=[9, 59]), 80, 3, 16),        # too few blocks, rows behind the last, narrow table
    (dict(counts=[], cached=[], new=[]), 5, 4, 16),                       # no sequence at all
    (dict(counts=[], cached=[], new=[]), 0, 1, 16),
    (dict(counts=[3, 2], cached=[1, 4], new=[6, 1]), 7, 5, 3),            # block size that is no power of two
    (dict(counts=[-4, 2, 3], cached=[-9, 3, 0], new=[-1, 4, 40]), 44, 9, 16),     # negative lengths count as 0
    (dict(counts=[4, 4], cached=[0, 0], new=[40, 40]), 50, 4, 16),        # more tokens than rows
]


@pytest.mark.parametrize("lens,total,width,block", MAPS)
def test_batch_maps(lens, total, width, block):
    ids = torch.randperm(100)[:sum(max(0, c) for c in lens["counts"])].to(torch.int32)
    args = [ids, *(torch.tensor(lens[k], dtype=torch.int32) for k in ("counts", "cached", "new"))]
    want = serving.batch_maps(*args, total, width, block_size=block, pad_block=777)
    got = serving.batch_maps(*(a.cuda() for a in args), total, width, block_size=block, pad_block=777)
    for name, a, b in zip(serving.BatchMaps._fields, got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b), name


@pytest.mark.parametrize("n,most", [(257, 40), (5000, 9), (16384, 3)])
def test_batch_maps_of_many_sequences(n, most):
    gen = torch.Generator().manual_seed(n)
    cached, new = (torch.randint(0, most, (n,), generator=gen) for _ in range(2))
    counts = (cached + new + 15) // 16 + torch.randint(0, 2, (n,), generator=gen)
    ids = torch.randint(0, 2**31 - 1, (int(counts.sum()),), generator=gen)
    total, width = int(new.sum()), int(counts.max()) + 1
    got = serving.batch_maps(*(_i32(t.tolist()) for t in (ids, counts, cached, new)), total, width, pad_block=3)
    # the same by whole-tensor operations in 64 bits
    seq = torch.repeat_interleave(torch.arange(n), new)
    at = cached[seq] + torch.arange(total) - (torch.cumsum(new, 0) - new)[seq]
    first = torch.cumsum(counts, 0) - counts
    assert torch.equal(got.positions.cpu().long(), at)
    assert torch.equal(got.slots.cpu(), ids[first[seq] + at // 16] * 16 + at % 16)              # block ids near 2^31: slots pass 32 bits
    column = torch.arange(width)
    tables = torch.where(column < counts[:, None], ids[(first[:, None] + column).clamp(max=ids.numel() - 1)], 3)
    assert torch.equal(got.tables.cpu().long(), tables)
    assert got.q_start.tolist() == [0] + torch.cumsum(new, 0).tolist() and got.context_lens.tolist() == (cached + new).tolist()


def test_batch_maps_survives_absurd_lengths_and_keeps_to_its_buffers():
    big = 2**31 - 1
    guard = 64
    kept, views = [], []
    for shape, dtype in (((4, 8), torch.int32), ((32,), torch.int32), ((32,), torch.int64), ((5,), torch.int32), ((4,), torch.int32)):
        flat = torch.full((math.prod(shape) + 2 * guard,), -5, dtype=dtype, device=_dev())
        kept.append(flat)
        views.append(flat[guard:guard + math.prod(shape)].view(shape))
    got = serving.batch_maps(_i32([5, 6, 7]), _i32([big, big, 2, -big]), _i32([big, 3, 0, 9]), _i32([big, 4, big, 1]), 32, 8, pad_block=1,
                             out=tuple(views))
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(got, views))
    assert got.positions.tolist() == [big] * 32                  # the first sequence's tokens sit at the largest position
    assert got.slots.tolist() == [1 * 16 + (big + j) % 16 for j in range(32)] and got.tables[0].tolist() == [5, 6, 7] + [1] * 5
    for flat, view in zip(kept, views):
        assert torch.all(flat[:guard] == -5) and torch.all(flat[guard + view.numel():] == -5)


def test_batch_maps_of_lengths_past_32_bits():
    big = 2**31 - 1
    args = ([5, 6], [1, 1], [big - 1, big], [3, big])
    got = serving.batch_maps(*map(_i32, args), 5, 1, pad_block=9)
    want = serving.batch_maps(*(_i32(a, "cpu") for a in args), 5, 1, pad_block=9)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_batch_maps_replayed_from_a_graph():
    ids, counts, cached, new = _i32(list(range(40))), _i32([10, 10, 10, 10]), _i32([3, 16, 31, 100]), _i32([5, 1, 2, 8])
    out = serving.batch_maps(ids, counts, cached, new, 16, 12, pad_block=99)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serving.batch_maps(ids, counts, cached, new, 16, 12, pad_block=99, out=out)
    cached.copy_(_i32([0, 1, 2, 3]))
    new.copy_(_i32([1, 1, 0, 12]))
    graph.replay()
    want = serving.batch_maps(ids.cpu(), counts.cpu(), cached.cpu(), new.cpu(), 16, 12, pad_block=99)
    for a, b in zip(out, want):
        assert torch.equal(a.cpu(), b)


_MAPS_OF_SIZES = """
import torch
from ajllm_b200.ops import serving
for n in (4089, 4090, 4095, 4096, 16384, 4095):
    ones = torch.ones(n, dtype=torch.int32, device="cuda")
    got = serving.batch_maps(torch.arange(n, dtype=torch.int32, device="cuda"), ones, ones - 1, ones, n, 1)
    assert torch.equal(got.slots, 16 * torch.arange(n, device="cuda")) and int(got.q_start[n]) == n, n
"""


def test_batch_maps_whose_lengths_just_fill_the_ordinary_shared_memory():
    """In a process that has made no larger call: 12 bytes per sequence and the kernel's static array pass 48 KB from 4090 on."""
    done = subprocess.run([sys.executable, "-c", _MAPS_OF_SIZES], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]


def test_batch_maps_of_large_and_small_batches_from_two_threads():
    failed = []

    def calls(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                ones = torch.ones(n, dtype=torch.int32, device=_dev())
                ids = torch.arange(n, dtype=torch.int32, device=_dev())
                for _ in range(200):
                    got = serving.batch_maps(ids, ones, ones - 1, ones, n, 1)
                assert torch.equal(got.slots, 16 * ids.long())
        except Exception as error:          # (an assertion in a thread would be lost)
            failed.append(error)

    threads = [threading.Thread(target=calls, args=(n,)) for n in (16384, 4200, 16384, 5000)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failed


# --------------------------------------------------------------------------------------------- attention


def _batch(heads, kv_heads, hd, q_len, prefix, suffixes, seed=0, poison=True):
    """Queries, caches, tables and lengths of sequences with a common prefix in shuffled blocks. With ``poison`` every
    cache slot that no sequence has written holds a NaN or an infinity."""
    gen = torch.Generator().manual_seed(seed)
    n, shared = len(suffixes), prefix // 16
    context = [prefix + s for s in suffixes]
    own = [(c + 15) // 16 - shared for c in context]
    order = torch.randperm(shared + sum(own) + 5, generator=gen)
    width = max(1, shared + max(own) + 1)
    tables = torch.full((n, width), int(order[-1]), dtype=torch.int64)
    tables[:, :shared] = order[:shared]
    cursor = shared
    for i, count in enumerate(own):
        tables[i, shared:shared + count] = order[cursor:cursor + count]
        cursor += count
    keys, values = (torch.randn(order.numel(), 16, kv_heads, hd, generator=gen) for _ in range(2))
    if prefix % 16:
        at = tables[:, shared]
        for cache in (keys, values):
            cache[at, :prefix % 16] = cache[at[0], :prefix % 16].clone()
    if poison:
        used = torch.zeros(order.numel(), 16, dtype=torch.bool)
        for i, c in enumerate(context):
            place = torch.arange(c)
            used[tables[i, place // 16], place % 16] = True
        keys[~used] = math.nan
        values[~used] = torch.tensor([math.inf, -math.inf, math.nan, 3e38])[torch.arange(int((~used).sum())) % 4][:, None, None]
    q = 1.5 * torch.randn(n * q_len, heads, hd, generator=gen)
    bf16 = [t.to(torch.bfloat16).cuda() for t in (q, keys, values)]
    return (*bf16, _i32(tables.tolist()), _i32(context))


def _oracle(q, keys, values, tables, context, q_len, scale=None):
    """``(out, sum of p |v|)`` in 64 bits, every sequence over its own blocks in order."""
    heads, hd = q.shape[1:]
    kv_heads = keys.shape[2]
    scale = scale or hd ** -0.5
    out, size = [], []
    for i, c in enumerate(context.tolist()):
        place = torch.arange(c, device=q.device)
        block = tables[i].long()[place // 16]
        k, v = (t[block, place % 16].double().repeat_interleave(heads // kv_heads, 1) for t in (keys, values))
        scores = torch.einsum("ihd,shd->ihs", q[i * q_len:(i + 1) * q_len].double(), k) * scale
        last = c - q_len + torch.arange(q_len, device=q.device)
        p = torch.softmax(scores.masked_fill(place > last[:, None, None], -math.inf), -1)
        out.append(torch.einsum("ihs,shd->ihd", p, v))
        size.append(torch.einsum("ihs,shd->ihd", p, v.abs()))
    return torch.cat(out), torch.cat(size)


def _check_attention(got, want, size):
    # probabilities and outputs are each rounded to bf16 once (half a step of sum p |v|, half a step of the output); the
    # rest is fp32: an exponent off by 1e-5 (128-term dot products of |s| < 100 and exp2's two steps) moves p by 1e-5
    bound = HALF_BF16 * (size + want.abs()) + 1e-4 * size + 1e-30
    worst = ((got.double() - want).abs() / bound).max()
    assert torch.isfinite(got).all() and float(worst) <= 1.0, float(worst)
    assert native.lib().ajb_check_status() == 0


SHAPES = [
    (8, 2, 128, 1, 512, [1, 17, 130, 500]),
    (4, 4, 64, 1, 16, [1]),                              # one sequence, one block
    (32, 8, 128, 1, 129, [1, 2, 64, 65, 200]),           # prefix ends one token into a block
    (32, 8, 64, 1, 4001, [3, 400]),
    (6, 2, 128, 1, 144, list(range(1, 51))),             # group of 3; more rows than a tile, tail tile
    (16, 2, 64, 1, 2048, [16, 48, 64, 80]),              # suffixes of whole blocks
    (8, 1, 128, 5, 333, [5, 6, 70]),                     # verification, 40 rows per sequence
    (16, 4, 128, 5, 100, [5, 130]),                      # verification, 20 rows (replicated variant)
    (128, 1, 64, 1, 260, [1, 90]),                       # as many query heads per KV head as a tile has rows
    (48, 1, 128, 3, 64, [3, 20]),                        # 144 rows: two chunks, the second partly filled
    (8, 2, 64, 61, 200, [61, 99]),                       # a chunk of a prompt, odd length
    (4, 2, 128, 1, 0, [1, 33, 700]),                     # nothing shared
    (4, 2, 128, 2, 15, [2, 33]),                         # a prefix shorter than a block
    (1, 1, 128, 1, 1024, [1] * 130),                     # one head: rows of a tile are all different sequences
]


@pytest.mark.parametrize("heads,kv_heads,hd,q_len,prefix,suffixes", SHAPES)
def test_shared_prefix_attention(heads, kv_heads, hd, q_len, prefix, suffixes):
    q, keys, values, tables, context = _batch(heads, kv_heads, hd, q_len, prefix, suffixes)
    got = serving.shared_prefix_attention(q, keys, values, tables, context, prefix, q_len=q_len)
    _check_attention(got, *_oracle(q, keys, values, tables, context, q_len))


@pytest.mark.parametrize("heads,kv_heads,hd,q_len,prefix,suffixes", [
    (32, 2, 128, 1, 300, list(range(1, 34))),            # 16 rows per sequence, so many pieces of the prefix
    (64, 2, 128, 1, 700, [1, 40, 7]),                    # 32 rows per sequence
    (20, 4, 128, 1, 513, [1, 5, 200, 16, 17, 3, 8]),     # 5 heads per KV head: pieces of 15 rows, the last one of 5
    (14, 2, 64, 2, 1000, [2, 30, 100]),                  # 14 rows per sequence: a piece of two tokens may span sequences
    (8, 8, 128, 5, 640, [5, 129, 6, 7]),                 # one head per KV head: pieces of 16 tokens out of 20
    (12, 4, 64, 7, 130, [7, 8, 300]),                    # 21 rows per sequence: pieces of 10 tokens out of 21
    (8, 2, 128, 1, 4096, [3, 900] * 12),                 # few long pieces
])
def test_prefixes_in_pieces_of_the_paged_launch(heads, kv_heads, hd, q_len, prefix, suffixes, monkeypatch):
    """The same through pieces of several sizes, whatever the plan would take, and through the prefix kernel."""
    q, keys, values, tables, context = _batch(heads, kv_heads, hd, q_len, prefix, suffixes)
    want = _oracle(q, keys, values, tables, context, q_len)
    group, tiles, rows = heads // kv_heads, -(-(prefix // 16) // 8), len(suffixes) * q_len * heads // kv_heads
    tokens = (16 if group * q_len <= 16 else 32) // group
    for pieces_of, ours, splits in ((tokens, 1, 1), (tokens, tiles, 3), (1, min(tiles, 2), 2), (0, 1, 1), (0, tiles, 2)):
        parts = splits + (2 * ours if pieces_of == 0 and rows <= 128 and ours < tiles else ours)
        monkeypatch.setattr(serving, "prefix_plan", lambda *a: (pieces_of, ours, splits, parts))
        _check_attention(serving.shared_prefix_attention(q, keys, values, tables, context, prefix, q_len=q_len), *want)


def test_shared_prefix_attention_with_large_scores_and_a_given_scale():
    """Scores of several hundred: the running maximum moves again and again, within the prefix and behind it."""
    q, keys, values, tables, context = _batch(8, 2, 128, 1, 640, [40, 300, 9], seed=3)
    ramp = torch.linspace(0.1, 3.0, keys.shape[0], device=_dev())[torch.randperm(keys.shape[0], device=_dev())]
    keys = (keys.float() * ramp[:, None, None, None]).to(torch.bfloat16)
    want, size = _oracle(q, keys, values, tables, context, 1, scale=1.0)
    got = serving.shared_prefix_attention(q, keys, values, tables, context, 640, scale=1.0)
    # products of |q k| up to 128 * 5 * 13 summed in fp32: the exponent is off by up to 128 * 2^-24 * 8e3 = 0.06
    bound = HALF_BF16 * (size + want.abs()) + 0.065 * 2 * size
    assert bool(((got.double() - want).abs() <= bound).all())
    assert native.lib().ajb_check_status() == 0


def test_scales_at_the_ends_of_their_range(monkeypatch):
    """With the smallest every visible key counts alike, with the largest only the best one does; beyond them calls are refused."""
    for batch, prefix in ((_batch(8, 2, 128, 1, 640, [40, 300, 9]), 640), (_batch(8, 2, 64, 1, 2048, [33] * 70), 2048)):
        q, keys, values, tables, context = batch
        want, size = _oracle(*batch, 1, scale=1e-30)
        _check_attention(serving.shared_prefix_attention(*batch, prefix, scale=1e-30), want, size)
        # scores are elements of the keys, exactly: those of up to 5 make exponents of 7000, off by 7000 * 2^-24 = 4e-4, the same for
        # every key that has the largest score (others have no weight: two bf16 numbers near 4 are 22 exponents apart)
        q.copy_(torch.eye(8, q.shape[2], device=_dev())[None].expand_as(q))
        want, size = _oracle(*batch, 1, scale=1e3)
        _check_attention(serving.shared_prefix_attention(*batch, prefix, scale=1e3), want, size)
    for fast in (native.fast, None):
        monkeypatch.setattr(native, "fast", fast)
        for scale in (1e-46, 1e-40, 1e39):
            with pytest.raises(ValueError, match="between"):
                serving.shared_prefix_attention(*batch, prefix, scale=scale)


def test_shared_prefix_attention_equals_paged_attention_closely():
    q, keys, values, tables, context = _batch(32, 8, 128, 1, 1024, [7, 260, 31], poison=False)
    a = serving.shared_prefix_attention(q, keys, values, tables, context, 1024)
    b = serving.paged_attention(q, keys, values, tables, None, None, [1] * 3, context.tolist())
    want, size = _oracle(q, keys, values, tables, context, 1)
    _check_attention(a, want, size)
    _check_attention(b, want, size)


def test_rows_without_a_key_are_zero():
    q, keys, values, tables, context = _batch(4, 2, 64, 1, 0, [5, 1, 40])
    context[1] = 0
    got = serving.shared_prefix_attention(q, keys, values, tables, context, 0)
    assert torch.count_nonzero(got[1]) == 0 and torch.count_nonzero(got[0]) > 0


@pytest.mark.parametrize("heads,kv_heads,hd,q_len,prefix,suffixes", [
    (8, 2, 128, 1, 512, [1, 17, 130, 500]),              # the prefix in pieces of the paged launch
    (32, 8, 64, 5, 2048, [5, 40] * 20),                  # the prefix kernel, two row tiles
    (32, 8, 128, 1, 4096, [3, 900] * 12),                # the prefix kernel or long pieces, many parts
    (48, 1, 128, 3, 64, [3, 20, 50]),                    # more than 32 rows per sequence
    (4, 2, 64, 1, 0, [1, 33, 700]),                      # nothing shared
])
def test_what_is_not_a_number_is_not_lost_between_the_parts(heads, kv_heads, hd, q_len, prefix, suffixes):
    """NaN in a query, in a visible key behind the prefix and in one of the prefix, and values whose weight is next to nothing:
    the rows that the definition gives are NaN, and no others change. ``paged_attention``, in parts or whole, does the same."""
    q, keys, values, tables, context = _batch(heads, kv_heads, hd, q_len, prefix, suffixes, poison=False)
    lens = context.tolist()

    def check():
        want, size = _oracle(q, keys, values, tables, context, q_len)
        for got in (serving.shared_prefix_attention(q, keys, values, tables, context, prefix, q_len=q_len),
                    *([serving.paged_attention(q, keys, values, tables, None, None, [q_len] * len(lens), lens)] if heads // kv_heads * q_len <= 64 else [])):
            assert torch.equal(got.isnan(), want.isnan())
            real = ~want.isnan()
            bound = HALF_BF16 * (size + want.abs()) + 1e-4 * size + 1e-30
            assert bool(((got.double() - want).abs() <= bound)[real].all())
        return want.isnan()

    assert not check().any()
    whole = q.clone()
    q[0, heads - 1, 3] = math.nan
    assert int(check().any(-1).sum()) == 1
    q.copy_(whole)
    last = lens[1] - q_len                              # position of the first new token of sequence 1
    block, offset = int(tables[1, last // 16]), last % 16
    kept = keys[block, offset, 0].clone()
    keys[block, offset, 0] = math.nan
    assert int(check().any(-1).sum()) == q_len * heads // kv_heads
    keys[block, offset, 0] = kept
    if prefix:
        block, kept = int(tables[0, prefix // 32]), keys[int(tables[0, prefix // 32]), 7, kv_heads - 1].clone()
        keys[block, 7, kv_heads - 1] = math.inf         # scores of both signs, or a NaN where a query's elements cancel
        q[:, -1] = q[:, -1].abs()                       # (the last head: all positive, a score of infinity)
        assert check()[:, -1].all()
        keys[block, 7, kv_heads - 1] = kept
        q.copy_(whole)
    assert native.lib().ajb_check_status() == 0


@pytest.mark.parametrize("q_len", [1, 20])
def test_values_of_visible_keys_count_whatever_their_weight(q_len):
    """A NaN value behind a prefix whose scores are 300 larger: its weight is 0 in fp32, 0 times NaN is NaN."""
    q, keys, values, tables, context = _batch(8, 2, 128, q_len, 512, [q_len, q_len + 30], poison=False)
    q[..., 0], keys[..., 0] = 200.0, 0.0
    shared = tables[0, :32].long()
    keys[shared, :, :, 0] = 20.0                        # 200 * 20 / sqrt(128) = 354 more for every key of the prefix
    last = int(context[1]) - q_len
    values[int(tables[1, last // 16]), last % 16, 1, 5] = math.nan
    got = serving.shared_prefix_attention(q, keys, values, tables, context, 512, q_len=q_len)
    want = torch.zeros_like(got, dtype=torch.bool)
    want[q_len:, 4:, 5] = True
    assert torch.equal(got.isnan(), want)


@pytest.mark.parametrize("q_len,prefix,suffixes", [(1, 512, [1, 17, 130]), (20, 512, [20, 33, 150]), (1, 0, [1, 33, 700]), (1, 2048, [9] * 90)])
def test_rows_of_scores_that_are_all_minus_infinity_are_zero(q_len, prefix, suffixes):
    """As in the CPU form."""
    q, keys, values, tables, context = _batch(8, 2, 128, q_len, prefix, suffixes, poison=False)
    keys.abs_().clamp_(min=2.0 ** -10)
    q[q_len, 2] = -math.inf
    got = serving.shared_prefix_attention(q, keys, values, tables, context, prefix, q_len=q_len)
    plain = serving.shared_prefix_attention(*(t.float().cpu() for t in (q, keys, values)), tables.cpu(), context.cpu(), prefix, q_len=q_len)
    assert torch.count_nonzero(got[q_len, 2]) == 0 and torch.count_nonzero(plain[q_len, 2]) == 0
    assert torch.isfinite(got).all() and torch.isfinite(plain).all()


def test_queries_read_in_place_from_packed_rows_and_results_into_a_given_tensor():
    q, keys, values, tables, context = _batch(8, 2, 128, 2, 200, [2, 50, 3])
    packed = torch.full((6, 12 * 128), math.nan, dtype=torch.bfloat16, device=_dev())
    packed[:, :1024] = q.view(6, 1024)
    out = torch.full((8, 8, 128), 7.0, dtype=torch.bfloat16, device=_dev())
    view, _, _ = (t for t in (packed[:, :1024].view(6, 8, 128), None, None))
    got = serving.shared_prefix_attention(view, keys, values, tables, context, 200, q_len=2, out=out[1:7])
    assert got.data_ptr() == out[1:].data_ptr() and torch.all(out[0] == 7) and torch.all(out[7] == 7)
    assert torch.equal(got, serving.shared_prefix_attention(q, keys, values, tables, context, 200, q_len=2))
    odd = torch.randn(6, 8, 130, device=_dev()).to(torch.bfloat16)[:, :, 1:129]          # rows that are not 16-byte aligned
    assert torch.equal(serving.shared_prefix_attention(odd, keys, values, tables, context, 200, q_len=2),
                       serving.shared_prefix_attention(odd.contiguous(), keys, values, tables, context, 200, q_len=2))


def test_two_captured_graphs_and_eager_calls_do_not_disturb_each_other():
    first = _batch(16, 4, 128, 1, 300, [3, 77, 12], seed=1)
    second = _batch(8, 2, 64, 4, 500, [4, 9], seed=2)
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for (q, keys, values, tables, context), prefix, q_len in ((first, 300, 1), (second, 500, 4)):
        serving.shared_prefix_attention(q, keys, values, tables, context, prefix, q_len=q_len)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(serving.shared_prefix_attention(q, keys, values, tables, context, prefix, q_len=q_len))
        graphs.append(graph)
    first[0].normal_()                           # replays read the inputs anew
    first[4].sub_(_i32([1, 5, 2]))
    for _ in range(3):
        graphs[0].replay()
        graphs[1].replay()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = serving.shared_prefix_attention(*first, 300)
    torch.cuda.current_stream().wait_stream(side)
    _check_attention(outs[0], *_oracle(*first, 1))
    _check_attention(outs[1], *_oracle(*second, 4))
    assert torch.equal(eager, outs[0])


@pytest.mark.parametrize("heads,kv_heads,hd,q_len,prefix,suffixes", [
    (32, 8, 128, 1, 1024, list(range(1, 150))),          # more pieces than run at once: which CTA takes which one varies
    (32, 8, 64, 5, 2048, [5, 40, 300] * 30),
    (8, 2, 64, 61, 200, [61, 99] * 8),
])
def test_the_same_call_repeats_itself_bit_for_bit(heads, kv_heads, hd, q_len, prefix, suffixes):
    batch = _batch(heads, kv_heads, hd, q_len, prefix, suffixes)
    lens = batch[4].tolist()
    calls = [lambda: serving.shared_prefix_attention(*batch, prefix, q_len=q_len)]
    if heads // kv_heads * q_len <= 64:
        calls.append(lambda: serving.paged_attention(*batch[:4], None, None, [q_len] * len(lens), lens))
    for call in calls:
        first = call()
        assert all(torch.equal(first, call()) for _ in range(10))


def test_tables_shorter_than_the_context_bound_what_is_read():
    """A context length beyond the block table (a caller's mistake that only the device sees) reads nothing behind it."""
    q, keys, values, tables, context = _batch(8, 2, 128, 1, 64, [100, 30], poison=False)
    context[0] = 10_000_000
    got = serving.shared_prefix_attention(q, keys, values, tables, context, 64)
    assert torch.isfinite(got).all() and native.lib().ajb_check_status() == 0


# --------------------------------------------------------------------------------------------- logits


def _logits_inputs(rows, vocab, dtype, width, biases, masked, seed=0):
    gen = torch.Generator().manual_seed(seed)
    kw = dict(history=torch.randint(-2, min(vocab + 3, 50), (rows, width), generator=gen).to(torch.int32),
              prompt_lens=torch.randint(0, width + 1, (rows,), generator=gen).to(torch.int32),
              history_lens=torch.randint(0, width + 1, (rows,), generator=gen).to(torch.int32),
              repetition=0.5 + torch.rand(rows, generator=gen), presence=torch.rand(rows, generator=gen) - 0.5,
              frequency=torch.rand(rows, generator=gen))
    if biases:
        kw["bias_ids"] = torch.randint(-1, min(vocab + 2, 40), (rows, biases), generator=gen).to(torch.int32)
        kw["bias_values"] = 3 * torch.randn(rows, biases, generator=gen)
    if masked:
        kw["token_mask"] = torch.randint(-2**31, 2**31 - 1, (rows, (vocab + 31) // 32), generator=gen).to(torch.int32)
    return (4 * torch.randn(rows, vocab, generator=gen)).to(dtype), kw


def _logits_oracle(logits, kw):
    """Token by token in 64 bits: ``(result, sum of the sizes that were added up)``."""
    x = logits.double()
    size = x.abs()
    rows, vocab = x.shape
    for r in range(rows):
        tokens = kw["history"][r, :int(kw["history_lens"][r])].tolist() if "history" in kw else []
        made = tokens[int(kw["prompt_lens"][r]):] if tokens else []
        for v in {t for t in tokens if 0 <= t < vocab}:
            f = float(kw["repetition"][r])
            x[r, v] = x[r, v] / f if x[r, v] > 0 else x[r, v] * f
            c = made.count(v)
            size[r, v] = x[r, v].abs() + abs(float(kw["frequency"][r])) * c + abs(float(kw["presence"][r]))
            x[r, v] -= float(kw["frequency"][r]) * c + (float(kw["presence"][r]) if c else 0.0)
        for v, b in zip(kw["bias_ids"][r].tolist(), kw["bias_values"][r].tolist()) if "bias_ids" in kw else ():
            if 0 <= v < vocab:
                x[r, v] += b
                size[r, v] += abs(b)
        if "token_mask" in kw:
            for v in range(vocab):
                if not (int(kw["token_mask"][r, v // 32]) >> (v % 32)) & 1:
                    x[r, v] = -math.inf
    return x, size


LOGITS = [
    (1, 1, torch.float32, 3, 0, False), (2, 33, torch.bfloat16, 9, 5, True), (3, 300, torch.bfloat16, 70, 40, True),
    (5, 8191, torch.float32, 600, 33, True), (2, 8195, torch.bfloat16, 64, 64, True), (1, 32000, torch.bfloat16, 40, 0, False),
    (2, 1030, torch.bfloat16, 0, 3, False), (4, 64, torch.float32, 1, 1, True),
]


@pytest.mark.parametrize("rows,vocab,dtype,width,biases,masked", LOGITS)
def test_process_logits(rows, vocab, dtype, width, biases, masked):
    logits, kw = _logits_inputs(rows, vocab, dtype, width, biases, masked)
    got = serving.process_logits(logits.cuda(), **{k: v.cuda() for k, v in kw.items()}).cpu()
    want, size = _logits_oracle(logits, kw)
    hidden = torch.isinf(want)
    assert torch.equal(torch.isinf(got) & (got < 0), hidden)
    # at most: quotient or product, frequency product, two differences, one sum per bias, each off by half a step
    bound = (4 + biases) * HALF_FP32 * size
    assert bool(((got.double() - want).abs()[~hidden] <= bound[~hidden]).all())
    assert torch.equal(got, serving.process_logits(logits, **kw))              # and the same fp32 steps as on the CPU


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_process_logits_of_strided_and_misaligned_rows(dtype, offset):
    logits, kw = _logits_inputs(7, 2051, dtype, 30, 9, True, seed=offset)
    wide = torch.full((7, 2100 + offset), math.nan, dtype=dtype)
    wide[:, offset:offset + 2051] = logits
    kw = {k: v.cuda() for k, v in kw.items()}
    got = serving.process_logits(wide.cuda()[:, offset:offset + 2051], **kw)
    assert torch.equal(got, serving.process_logits(logits.cuda(), **kw))
    kept = torch.full((7 * 2051 + 20,), 5.0, device=_dev())
    again = serving.process_logits(logits.cuda(), **kw, out=kept[8:8 + 7 * 2051].view(7, 2051))
    assert torch.equal(got, again) and torch.all(kept[:8] == 5) and torch.all(kept[8 + 7 * 2051:] == 5)
    transposed = logits.t().contiguous().cuda().t()
    assert torch.equal(got, serving.process_logits(transposed, **kw))


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_subnormal_logits_penalties_and_biases_are_not_taken_for_zero(rows, dtype):
    """One launch and two; every kind of step with operands or results below the smallest normal number."""
    vocab = 32_000
    small = torch.tensor([1e-40, -1e-40, 1e-44, -1e-44, 1.3e-38, -1.3e-38, 0.0, -0.0, 1e-3, -2.0])
    logits = small.repeat(vocab // 10).expand(rows, -1).to(dtype).contiguous()
    history = torch.arange(200, dtype=torch.int32).repeat(rows, 1)
    lens = torch.full((rows,), 200, dtype=torch.int32)
    row = torch.arange(rows)
    kw = dict(history=history, prompt_lens=lens // 2, history_lens=lens, repetition=torch.tensor([1.7, 0.6, 1e-3])[row % 3],
              presence=torch.tensor([0.0, 3e-41, -2e-38])[row % 3], frequency=torch.tensor([1e-41, 0.0, 1.2e-38])[row % 3],
              bias_ids=torch.arange(150, 250, dtype=torch.int32).repeat(rows, 1), bias_values=torch.tensor([5e-41, -1e-38]).repeat(50).repeat(rows, 1))
    assert (rows * vocab >= 1 << 23) == (rows == 300)
    got = serving.process_logits(logits.cuda(), **{name: t.cuda() for name, t in kw.items()}).cpu()
    want = serving.process_logits(logits, **kw)
    assert torch.equal(got.view(torch.int32), want.view(torch.int32))
    # subnormal are 1e-40 and, in fp32, 1e-44 (bf16 ends at 9e-41), with both signs: at least 2 in 10, but for the 250 mended tokens
    assert int(((want != 0) & (want.abs() < 2.0 ** -126)).sum()) >= rows * (vocab - 250) // 10 * 2


def test_masked_places_hide_whatever_is_in_them_and_open_ones_keep_it():
    values = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min, 1.0, 0.0, -0.0, 2.0])
    logits = values.repeat(3, 8)
    mask = torch.tensor([[0, 0], [-1, -1], [0b11110000, 0]], dtype=torch.int32)
    got = serving.process_logits(logits.cuda(), token_mask=mask.cuda()).cpu()
    assert torch.all(got[0] == -math.inf)                               # nothing left
    assert torch.equal(got[1].view(torch.int32), logits[1].view(torch.int32))
    assert torch.all(got[2, :4] == -math.inf) and got[2, 4:8].tolist() == [1.0, 0.0, 0.0, 2.0] and torch.all(got[2, 8:] == -math.inf)


def test_the_same_token_many_times():
    """A history and a bias list that hold one token only: every thread of the kernel meets on it."""
    logits = torch.ones(2, 5000, device=_dev())
    history = torch.full((2, 4096), 4321, dtype=torch.int32, device=_dev())
    lens = _i32([4096, 4095])
    ids = torch.full((2, 200), 4321, dtype=torch.int32, device=_dev())
    bias = torch.full((2, 200), 0.25, device=_dev())
    got = serving.process_logits(logits, history=history, prompt_lens=_i32([96, 4095]), history_lens=lens,
                                 repetition=torch.full((2,), 2.0, device=_dev()), frequency=torch.full((2,), 0.125, device=_dev()),
                                 presence=torch.full((2,), 0.5, device=_dev()), bias_ids=ids, bias_values=bias)
    assert got[:, 4321].tolist() == [0.5 - 500 - 0.5 + 50, 0.5 + 50]
    got[:, 4321] = 1
    assert torch.all(got == 1)


def test_logits_maps_and_attention_replayed_together():
    """One decoding step as a server runs it: maps, cache write, attention behind the prefix, logits, sampler, captured
    once and replayed with other lengths."""
    torch.manual_seed(0)
    heads, kv_heads, hd, prefix, n, vocab = 8, 2, 128, 160, 3, 500
    _, keys, values, tables, _ = _batch(heads, kv_heads, hd, 1, prefix, [40, 40, 40], seed=5, poison=False)
    ids, counts = tables[:, :13].reshape(-1).contiguous(), _i32([13] * n)
    cached, new = _i32([prefix + 3, prefix + 15, prefix + 38]), _i32([1] * n)
    q, k, v = (torch.randn(n, h, hd, device=_dev()).to(torch.bfloat16) for h in (heads, kv_heads, kv_heads))
    head = (0.05 * torch.randn(vocab, heads * hd, device=_dev())).to(torch.bfloat16)
    history, lens = torch.randint(0, vocab, (n, 64), device=_dev(), dtype=torch.int32), _i32([10, 64, 33])
    penalty = torch.full((n,), 1.3, device=_dev())
    mask = torch.randint(-2**31, 2**31 - 1, (n, (vocab + 31) // 32), device=_dev()).to(torch.int32)
    zeros, ones = torch.zeros(n, device=_dev()), torch.ones(n, device=_dev())
    seeds = torch.arange(n, device=_dev())

    def step():
        maps = serving.batch_maps(ids, counts, cached, new, n, 13)
        keys.view(-1, kv_heads, hd).index_copy_(0, maps.slots, k)
        values.view(-1, kv_heads, hd).index_copy_(0, maps.slots, v)
        attended = serving.shared_prefix_attention(q, keys, values, maps.tables, maps.context_lens, prefix)
        raw = attended.view(n, -1) @ head.t()
        logits = serving.process_logits(raw, history=history, prompt_lens=lens // 2, history_lens=lens, repetition=penalty, token_mask=mask)
        return maps, attended, raw, logits, serving.sample_rows(logits, zeros, ones, seeds, seeds)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        maps, attended, raw, logits, tokens = step()
    cached.copy_(_i32([prefix, prefix + 31, prefix + 32]))
    graph.replay()
    assert maps.context_lens.tolist() == [prefix + 1, prefix + 32, prefix + 33]
    _check_attention(attended, *_oracle(q, keys, values, maps.tables, maps.context_lens, 1))
    want = reference.process_logits(raw.cpu(), history.cpu(), (lens // 2).cpu(), lens.cpu(), penalty.cpu(), token_mask=mask.cpu())
    assert torch.equal(logits.cpu(), want) and tokens.tolist() == want.argmax(-1).tolist()


def test_history_longer_than_a_16_bit_count():
    """40000 repeats of two tokens: counts need more than 15 bits."""
    rows, vocab, width = 2, 9000, 40000
    history = torch.full((rows, width), 8500, dtype=torch.int32, device=_dev())
    history[:, ::4] = 3
    kw = dict(prompt_lens=_i32([0, 39000]), history_lens=_i32([width, width]), frequency=torch.full((rows,), 2.0 ** -10, device=_dev()))
    got = serving.process_logits(torch.zeros(rows, vocab, device=_dev()), history=history, **kw)
    assert got[:, 3].tolist() == [-10000 / 1024, -250 / 1024] and got[:, 8500].tolist() == [-30000 / 1024, -750 / 1024]
    got[:, [3, 8500]] = 0
    assert torch.count_nonzero(got) == 0


@pytest.mark.parametrize("rows,vocab,dtype,width,biases,masked,offset", [
    (70, 128256, torch.bfloat16, 700, 40, True, 0), (300, 31999, torch.float32, 5000, 3, True, 1), (90, 100001, torch.bfloat16, 4096, 0, False, 0),
    (530, 16384, torch.float32, 33, 70, True, 0), (66, 128256, torch.bfloat16, 0, 5, True, 3), (65, 131072, torch.bfloat16, 1, 0, False, 0)])
def test_process_logits_of_many_rows(rows, vocab, dtype, width, biases, masked, offset):
    """Sizes at which the rows are streamed by one launch and mended by another; histories longer than a CTA holds."""
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    kw = dict(device="cuda", generator=gen)
    wide = (4 * torch.randn(rows, vocab + 5, **kw)).to(dtype)
    logits = wide[:, offset:offset + vocab]
    args = {}
    if width:
        ids = (vocab ** torch.rand(rows, width, **kw) - 1).to(torch.int32)
        ids[torch.rand(rows, width, **kw) < 0.02] = vocab + 7
        args = dict(history=ids, prompt_lens=torch.randint(0, width + 1, (rows,), **kw).int(), history_lens=torch.randint(0, width + 1, (rows,), **kw).int(),
                    repetition=0.7 + torch.rand(rows, **kw), presence=torch.rand(rows, **kw), frequency=torch.rand(rows, **kw))
    if biases:
        args.update(bias_ids=torch.randint(-3, vocab + 3, (rows, biases), **kw).int(), bias_values=torch.randn(rows, biases, **kw))
        args["bias_ids"][:, biases // 2:] = args["bias_ids"][:, :biases - biases // 2]             # every token twice
    if masked:
        args["token_mask"] = torch.randint(-2**31, 2**31 - 1, (rows, (vocab + 31) // 32), **kw).int()
    assert rows * vocab >= 1 << 23
    got = serving.process_logits(logits, **args)
    want = reference.process_logits(logits, **args)               # the same fp32 steps, whole rows at a time
    assert torch.equal(got, want)
    assert torch.equal(got, serving.process_logits(logits.contiguous(), **args))


# ----------------------------------------------------------------------------- the serving engine

ENGINE_CFG = {"name": "s", "context_length": 512, "d_model": 512, "num_layers": 2, "num_heads": 4, "num_kv_heads": 2,
              "d_ff": 1408, "init": {"type": "normal", "std": 0.05}}


@pytest.fixture(scope="module")
def engine_model():
    from ajllm_b200.models import build_model
    torch.manual_seed(0)
    return build_model(ENGINE_CFG, 1000).to(device=torch.device("cuda", 0), dtype=torch.bfloat16)


def _engine_prompts():
    gen = torch.Generator().manual_seed(3)
    head = torch.randint(0, 1000, (150,), generator=gen).tolist()
    return head, [head + torch.randint(0, 1000, (n,), generator=gen).tolist() for n in (5, 40, 1, 130, 17, 64, 9)]


@pytest.mark.parametrize("graphs", ["1", "0"])
@pytest.mark.parametrize("count", [2, 7])
def test_runner_steps_behind_a_prefix(engine_model, monkeypatch, graphs, count):
    """Prefill and decoding steps behind a shared prefix against the model run on each whole sequence."""
    from ajllm_b200.engine import LLMEngine
    from ajllm_b200.engine.model_runner import RunItem
    monkeypatch.setenv("AJB_DECODE_GRAPHS", graphs)
    head, prompts = _engine_prompts()
    engine = LLMEngine(engine_model, num_blocks=256)
    assert engine.runner.use_graphs == (graphs == "1")
    assert engine.share_prefix(head) == 144
    parent = engine.scheduler.prefix[0]
    sequences = [list(p) for p in prompts[:count]]
    for i in range(count):
        engine.cache.fork(parent, i)
    calls = []
    real = serving.shared_prefix_attention
    monkeypatch.setattr(serving, "shared_prefix_attention", lambda *a, **k: calls.append(1) or real(*a, **k))
    logits = engine.runner.forward([RunItem(i, s[144:], 1) for i, s in enumerate(sequences)])
    assert not calls                                        # ragged: every sequence reads its own context
    for step in range(3):
        for i, sequence in enumerate(sequences):
            with torch.no_grad():
                want = engine_model(torch.tensor([sequence], device=logits.device))[0, -1].float()
            assert float((logits[i] - want).abs().max()) < 0.08 * float(want.abs().max())
            sequence.append(int(want.argmax()))
        logits = engine.runner.forward([RunItem(i, s[-1:], 1) for i, s in enumerate(sequences)])
    assert calls
    before = len(engine.runner._graphs)
    engine.release_prefix()
    assert len(engine.runner._graphs) == (before - 1 if graphs == "1" else 0)
    logits = engine.runner.forward([RunItem(i, [1], 1) for i in range(count)])       # the blocks outlive the prefix's own hold
    with torch.no_grad():
        want = engine_model(torch.tensor([sequences[0] + [1]], device=logits.device))[0, -1].float()
    assert float((logits[0] - want).abs().max()) < 0.08 * float(want.abs().max())
    assert native.lib().ajb_check_status() == 0


def test_engine_serves_requests_behind_a_prefix(engine_model):
    from ajllm_b200.engine import LLMEngine, SamplingParams
    head, prompts = _engine_prompts()
    params = SamplingParams(12, 0.0, None)
    plain = LLMEngine(engine_model, num_blocks=256, max_num_seqs=4).generate(prompts, params)
    engine = LLMEngine(engine_model, num_blocks=256, max_num_seqs=4)
    engine.share_prefix(head)
    graphs = engine.warm_up()
    outs = engine.generate(prompts, params)
    assert len(engine.runner._graphs) == graphs == 5           # 1, 2, 4 sequences, and 2 and 4 behind the prefix
    # The logits are bf16: two evaluations that sum in another order can round a logit to neighbouring values, one step of
    # 2^-8 to 2^-7 of it apart, so two logits that differ by two steps of the larger at most can change places. The first
    # token that differs from the plain engine's has to be such a case (what follows it then differs for good).
    for a, b in zip(plain, outs):
        first = next((i for i, (x, y) in enumerate(zip(a.output, b.output)) if x != y), None)
        if first is not None:
            with torch.no_grad():
                logits = engine_model(torch.tensor([a.prompt + a.output[:first]], device=_dev()))[0, -1].float()
            one, other = float(logits[a.output[first]]), float(logits[b.output[first]])
            assert abs(one - other) <= 2 * 2.0 ** -7 * max(abs(one), abs(other))
    assert engine.cache.allocator.free_blocks == 256 - 9 - 1
    assert native.lib().ajb_check_status() == 0


def test_engine_processes_logits(engine_model):
    """Penalties, biases and masks of a changing batch: every greedy token is the best of the formula on the model's logits."""
    from ajllm_b200.engine import LLMEngine, SamplingParams
    head, prompts = _engine_prompts()
    words = torch.zeros(32, dtype=torch.int32)
    words[5] = 0b1111
    params = [SamplingParams(9, 0.0, None, repetition_penalty=1.3), SamplingParams(5, 0.0, None, frequency_penalty=2.0, presence_penalty=0.5),
              SamplingParams(9, 0.0, None, token_mask=lambda output: words if len(output) < 4 else torch.zeros_like(words)),
              SamplingParams(7, 0.0, None, logit_bias={3: 100.0}, frequency_penalty=30.0), SamplingParams(9, 0.0, None), None, None]
    engine = LLMEngine(engine_model, num_blocks=256, max_num_seqs=3)
    engine.share_prefix(head)
    outs = engine.generate(prompts[:5], params[:5])
    assert [len(o.output) for o in outs] == [9, 5, 4, 7, 9] and outs[2].finish_reason == "mask"
    assert all(160 <= token < 164 for token in outs[2].output)
    assert outs[3].output[:3] == [3, 3, 3] and outs[3].output != [3] * 7
    for prompt, p, out in zip(prompts[:2], params[:2], outs[:2]):
        tokens = list(prompt)
        for token in out.output:
            with torch.no_grad():
                x = engine_model(torch.tensor([tokens], device=torch.device("cuda", 0)))[0, -1:].float().cpu()
            one = lambda v: torch.tensor([v])
            want = reference.process_logits(x, torch.tensor([tokens]).int(), one(len(prompt)).int(), one(len(tokens)).int(), one(p.repetition_penalty),
                                            one(p.presence_penalty), one(p.frequency_penalty))[0]
            assert float(want[token]) > float(want.max()) - 0.08 * float(x.abs().max())      # as far as the forwards may differ
            tokens.append(token)
    assert native.lib().ajb_check_status() == 0


# --------------------------------------------------------------------------------------------- limits and refusals


@pytest.mark.parametrize("q_len,count", [(1, 3), (1, 70), (20, 3)])
def test_cache_blocks_past_32_bits_and_table_entries_behind_the_context(q_len, count):
    """The last blocks of caches of 2.3e9 elements; whatever the tables hold behind a context is not looked up."""
    prefix, kv_heads, hd = 160, 8, 128
    suffixes = [q_len + (7 * i) % 50 for i in range(count)]
    q, keys, values, tables, context = _batch(16, kv_heads, hd, q_len, prefix, suffixes)
    want = _oracle(q, keys, values, tables, context, q_len)
    blocks = 140_000
    far = [torch.empty(blocks, 16, kv_heads, hd, dtype=torch.bfloat16, device=_dev()) for _ in range(2)]
    first = blocks - keys.shape[0]
    for cache, near in zip(far, (keys, values)):
        cache[first:] = near
    wide = torch.full((count, tables.shape[1] + 9), 2**31 - 1, dtype=torch.int32, device=_dev())
    wide[:, 1::2] = -7
    for i, length in enumerate(context.tolist()):
        wide[i, :(length + 15) // 16] = tables[i, :(length + 15) // 16] + first
    _check_attention(serving.shared_prefix_attention(q, *far, wide, context, prefix, q_len=q_len), *want)


def test_logits_past_32_bits():
    rows, vocab = 16_800, 128_256                        # 2.15e9 logits
    logits = torch.empty(rows, vocab, dtype=torch.bfloat16, device=_dev())
    checked = [0, 1, 16_743, 16_744, rows - 1]           # 2^31 lies in row 16743
    logits[checked] = torch.randn(len(checked), vocab, dtype=torch.bfloat16, device=_dev(), generator=torch.Generator(_dev()).manual_seed(0))
    history = torch.randint(0, vocab, (rows, 33), dtype=torch.int32, device=_dev())
    lens = torch.full((rows,), 33, dtype=torch.int32, device=_dev())
    kw = dict(history=history, prompt_lens=lens // 2, history_lens=lens, presence=torch.full((rows,), 0.5, device=_dev()),
              bias_ids=history[:, :3].contiguous(), bias_values=torch.ones(rows, 3, device=_dev()),
              token_mask=torch.randint(-2**31, 2**31 - 1, (rows, vocab // 32), dtype=torch.int32, device=_dev()))
    got = serving.process_logits(logits, **kw)
    want = serving.process_logits(logits[checked], **{k: v[checked] for k, v in kw.items()})       # few rows, small offsets
    assert torch.equal(got[checked], want)
    plain = reference.process_logits(logits[checked].cpu(), *(None if v is None else v[checked].cpu() for v in (
        kw["history"], kw["prompt_lens"], kw["history_lens"], None, kw["presence"], None, kw["bias_ids"], kw["bias_values"], kw["token_mask"])))
    assert torch.equal(want.cpu(), plain)


def test_many_rows_replayed_from_a_graph_and_calls_on_two_streams():
    """The two-launch form captured and replayed with other inputs, and beside calls on another stream."""
    def on_gpu(logits, kw):
        return logits.cuda(), {name: t.cuda() for name, t in kw.items()}

    logits, kw = on_gpu(*_logits_inputs(300, 32_000, torch.bfloat16, 40, 5, True))
    other, other_kw = on_gpu(*_logits_inputs(280, 31_999, torch.float32, 77, 3, True, seed=1))
    want_other = serving.process_logits(other, **other_kw)
    want = serving.process_logits(logits, **kw)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        serving.process_logits(logits, **kw, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    found = []
    for _ in range(5):
        out.zero_()
        graph.replay()
        with torch.cuda.stream(side):
            found.append(serving.process_logits(other, **other_kw))
    torch.cuda.synchronize()
    assert torch.equal(out, want) and all(torch.equal(f, want_other) for f in found)
    logits.copy_(logits.flip(0))
    kw["history"].copy_(kw["history"].flip(1))
    graph.replay()
    assert torch.equal(out, serving.process_logits(logits, **kw))


def test_attention_calls_on_two_streams():
    few = _batch(8, 2, 128, 1, 512, [1, 17, 130, 500])
    many = _batch(32, 8, 128, 1, 2048, list(range(1, 100)))
    calls = [(b, p, _oracle(*b, 1)) for b, p in ((few, 512), (many, 2048))]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    found = [[], []]
    for _ in range(4):
        for i, (batch, prefix, _) in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                found[i].append(serving.shared_prefix_attention(*batch, prefix))
    torch.cuda.synchronize()
    for results, (_, _, want) in zip(found, calls):
        for got in results:
            _check_attention(got, *want)


def test_results_that_cannot_be_written_are_refused():
    q, keys, values, tables, context = _batch(8, 2, 128, 1, 64, [3, 4])
    flat = torch.empty(q.numel() + 8, dtype=torch.bfloat16, device=_dev())
    with pytest.raises(RuntimeError, match="aligned"):
        serving.shared_prefix_attention(q, keys, values, tables, context, 64, out=flat[1:1 + q.numel()].view(q.shape))
    serving.shared_prefix_attention(q, keys, values, tables, context, 64, out=flat[8:].view(q.shape))
    for out in (q, values.flatten()[:q.numel()].view(q.shape)):
        with pytest.raises(ValueError, match="overlap"):
            serving.shared_prefix_attention(q, keys, values, tables, context, 64, out=out)
    ids, counts, cached, new = _i32([3, 4]), _i32([1, 1]), _i32([2, 0]), _i32([1, 1])
    good = serving.batch_maps(ids, counts, cached, new, 2, 2)
    for out in (good._replace(context_lens=cached), good._replace(q_start=good.tables.flatten()[:3])):
        with pytest.raises(RuntimeError, match="overlap"):
            serving.batch_maps(ids, counts, cached, new, 2, 2, out=out)
    with pytest.raises(RuntimeError, match="aligned"):
        serving.batch_maps(ids, counts, cached, new, 2, 2, out=good._replace(positions=torch.zeros(3, dtype=torch.int32, device=_dev())[1:]))
    logits = torch.zeros(2, 64, device=_dev())
    mask = torch.zeros(128, device=_dev())
    with pytest.raises(ValueError, match="overlap"):
        serving.process_logits(logits, token_mask=mask.view(torch.int32)[:4].view(2, 2), out=mask.view(2, 64))
    for wrong in (torch.float16, torch.float32):
        with pytest.raises(TypeError):
            serving.shared_prefix_attention(q.to(wrong), keys.to(wrong), values.to(wrong), tables, context, 64)
    with pytest.raises((ValueError, TypeError)):
        serving.shared_prefix_attention(q, keys, values, tables.cpu(), context, 64)
    with pytest.raises(RuntimeError, match="block size"):
        serving.shared_prefix_attention(q, keys.view(-1, 8, 2, 128), values.view(-1, 8, 2, 128), tables, context, 16)


def test_infinite_penalties_leave_other_tokens_alone():
    logits = torch.randn(2, 50, device=_dev())
    kw = dict(history=_i32([[3, 4, 5], [6, 7, 8]]), prompt_lens=_i32([2, 3]), history_lens=_i32([3, 3]),
              frequency=torch.tensor([math.inf, math.inf], device=_dev()))
    got = serving.process_logits(logits, **kw).cpu()
    want = reference.process_logits(logits.cpu(), *(kw[k].cpu() for k in ("history", "prompt_lens", "history_lens")), frequency=kw["frequency"].cpu())
    assert torch.equal(got, want) and torch.isinf(got).sum() == 1 and not torch.isnan(got).any()


@pytest.mark.parametrize("width", [9, 5000])
@pytest.mark.parametrize("rows,vocab", [(3, 1000), (270, 32_003)])
def test_ids_outside_the_vocabulary_are_skipped(rows, vocab, width):
    """Whatever they are, in either form and with histories of either size."""
    logits = torch.randn(rows, vocab, device=_dev())
    outside = torch.tensor([-1, -2, -3, -17, -vocab, vocab, vocab + 1, 2**31 - 1, -2**31], dtype=torch.int32)
    history = outside.repeat(rows, width // 9 + 1)[:, :width].contiguous().cuda()
    history[:, 4] = 2
    lens = torch.full((rows,), width, dtype=torch.int32, device=_dev())
    got = serving.process_logits(logits, history=history, prompt_lens=lens - width, history_lens=lens, presence=torch.ones(rows, device=_dev()),
                                 bias_ids=outside.repeat(rows, 1).cuda(), bias_values=torch.ones(rows, 9, device=_dev()))
    want = logits.clone()
    want[:, 2] -= 1.0
    assert torch.equal(got, want)


# --------------------------------------------------------------------------------------------- the extension that makes the calls


def _ordinary_calls():
    maps = (_i32([3, 4, 5]), _i32([1, 2]), _i32([2, 17]), _i32([1, 9]), 12, 4)
    attention = (*_batch(8, 2, 128, 1, 96, [3, 40]), 96)
    logits, kw = _logits_inputs(3, 300, torch.bfloat16, 7, 4, True)
    return [(serving.batch_maps, maps, dict(pad_block=1)), (serving.shared_prefix_attention, attention, dict(scale=0.1)),
            (serving.shared_prefix_attention, attention, dict(max_context=200)),
            (serving.process_logits, (logits.cuda(),), {name: t.cuda() for name, t in kw.items()})]


def test_both_ways_to_call_give_the_same(monkeypatch):
    """The extension, and what takes over where it does not apply: the same results, bit for bit, and launches counted alike."""
    assert native.fast is not None
    found = []
    for fast in (native.fast, None):
        monkeypatch.setattr(native, "fast", fast)
        for fn, args, kw in _ordinary_calls():
            before = native.launch_count
            got = fn(*args, **kw)
            found.append([*(got if isinstance(got, tuple) else [got]), native.launch_count - before])
    half = len(found) // 2
    for a, b in zip(found[:half], found[half:]):
        assert a[-1] == b[-1] and all(torch.equal(x, y) for x, y in zip(a[:-1], b[:-1]))


def test_ordinary_calls_go_through_the_extension(monkeypatch):
    monkeypatch.setattr(native, "call_packed", lambda *a: pytest.fail("the call was not taken"))
    for fn, args, kw in _ordinary_calls():
        fn(*args, **kw)
    out = serving.batch_maps(_i32([3]), _i32([1]), _i32([2]), _i32([1]), 1, 1)
    assert isinstance(out, serving.BatchMaps)
    again = serving.batch_maps(_i32([4]), _i32([1]), _i32([2]), _i32([1]), 1, 1, out=tuple(out))
    assert isinstance(again, serving.BatchMaps) and again.tables is out.tables and out.tables.tolist() == [[4]]


def test_contexts_that_grow_by_a_token_per_step_keep_their_plan(monkeypatch):
    q, keys, values, tables, context = _batch(8, 2, 128, 1, 512, [200, 300, 600], poison=False)
    for fast in (native.fast, None):
        monkeypatch.setattr(native, "fast", fast)
        serving.prefix_plan.cache_clear()
        for most in range(700, 956):                    # 2 tiles of 128 keys
            serving.shared_prefix_attention(q, keys, values, tables, context, 512, max_context=most)
        assert serving.prefix_plan.cache_info().misses <= 3


def test_calls_that_the_extension_leaves_alone():
    logits, kw = _logits_inputs(3, 300, torch.bfloat16, 7, 4, True)
    logits, kw = logits.cuda(), {name: t.cuda() for name, t in kw.items()}
    want = serving.process_logits(logits, **kw)
    assert torch.equal(serving.process_logits(torch.nn.Parameter(logits), **kw), want)                  # not a plain tensor
    assert torch.equal(serving.process_logits(logits.t().contiguous().t(), **kw), want)                 # columns next to one another
    q, keys, values, tables, context = _batch(8, 2, 128, 1, 96, [3, 40])
    want = serving.shared_prefix_attention(q, keys, values, tables, context, 96)
    wide = torch.zeros(2, 8, 160, dtype=torch.bfloat16, device=_dev())
    wide[..., 5:133] = q
    assert torch.equal(serving.shared_prefix_attention(wide[..., 5:133], keys, values, tables, context, 96), want)
    assert torch.equal(serving.shared_prefix_attention(q, keys, values, tables, context, 96, scale=torch.tensor(128 ** -0.5).item()), want)
    assert serving.shared_prefix_attention(q[:0], keys, values, tables[:0], context[:0], 96).shape == (0, 8, 128)
    assert serving.process_logits(logits[:0]).shape == (0, 300)


def test_a_result_that_does_not_fit_the_device_is_an_exception():
    row = torch.zeros(1, 1 << 20, device=_dev())
    with pytest.raises(torch.OutOfMemoryError):
        serving.process_logits(row.expand(300_000, -1))                    # 1.2 TB of results
    assert torch.equal(serving.process_logits(row), row)


# --------------------------------------------------------------------------------------------- launches that start early


def _slow_copies(pairs):
    """Writes every ``src`` into its ``dst`` behind a product that takes a while, the last write directly in front of what follows."""
    a = torch.full((4096, 4096), 1e-4, device=_dev(), dtype=torch.bfloat16)
    for dst, src in pairs:
        late = (a @ a).sum() * 0
        dst.copy_(src + late.to(src.dtype))


@pytest.mark.parametrize("captured", [False, True])
def test_inputs_written_directly_in_front_of_a_call_are_the_ones_it_reads(captured):
    """Each operator behind a launch that writes its inputs late, and in front of one that overwrites them."""
    logits, kw = _logits_inputs(5, 3000, torch.bfloat16, 40, 5, True)
    many, many_kw = _logits_inputs(300, 32_000, torch.bfloat16, 40, 5, True)
    few = _batch(8, 2, 128, 1, 512, [1, 17, 130, 500])
    rows = _batch(32, 8, 128, 1, 2048, list(range(1, 100)))
    maps = [_i32([3, 4, 5, 6]), _i32([1, 3]), _i32([2, 17]), _i32([1, 9])]

    def move(tensors):
        return [t.cuda() for t in tensors]

    cases = []
    for fn, given in ((lambda x, *t: serving.process_logits(x, **dict(zip(kw, t))), move([logits, *kw.values()])),
                      (lambda x, *t: serving.process_logits(x, **dict(zip(many_kw, t))), move([many, *many_kw.values()])),
                      (lambda *t: serving.shared_prefix_attention(*t, 512), list(few)),
                      (lambda *t: serving.shared_prefix_attention(*t, 2048), list(rows)),
                      (lambda *t: serving.batch_maps(*t, 12, 4, pad_block=1), maps)):
        want = fn(*given)
        torch.cuda.synchronize()
        cases.append((fn, given, [t.clone() for t in given], want if isinstance(want, tuple) else (want,)))

    def run():
        found = []
        for fn, given, kept, _ in cases:
            _slow_copies(zip(given, kept))
            got = fn(*given)
            for t in given:
                t.zero_()
            found.append(got if isinstance(got, tuple) else (got,))
        # and one behind another, each reading what the one in front of it has written
        _slow_copies([(cases[0][1][0], cases[0][2][0])])
        once = serving.process_logits(cases[0][1][0])
        found.append((serving.process_logits(serving.process_logits(once)),))
        return found

    for _, given, _, _ in cases:
        for t in given:
            t.zero_()
    if captured:
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            found = run()
        graph.replay()
        graph.replay()
    else:
        found = run()
    torch.cuda.synchronize()
    for got, (_, _, _, want) in zip(found, cases):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(found[-1][0], cases[0][2][0].float())


@pytest.mark.parametrize("captured", [False, True])
def test_calls_behind_two_streams(captured):
    """A call that follows work of its own stream and, through an event, of another one waits for both."""
    ids, counts, cached, new = maps = [_i32([3, 4, 5, 6]), _i32([1, 3]), _i32([2, 17]), _i32([1, 9])]
    kept = [t.clone() for t in maps]
    want = serving.batch_maps(*maps, 12, 4, pad_block=1)
    side = torch.cuda.Stream()

    def run():
        main = torch.cuda.current_stream()
        for t in maps:
            t.zero_()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            _slow_copies([(cached, kept[2]), (ids, kept[0])])
        new.copy_(kept[3])
        counts.copy_(kept[1])
        main.wait_stream(side)
        return serving.batch_maps(*maps, 12, 4, pad_block=1)

    if captured:
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        graph.replay()
    else:
        got = run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_runner_takes_a_step_of_too_many_sequences_in_parts(engine_model, monkeypatch):
    from ajllm_b200.engine import LLMEngine
    from ajllm_b200.engine.model_runner import ModelRunner, RunItem
    _, prompts = _engine_prompts()
    items = [RunItem(i, p, 1 + i % 2) for i, p in enumerate(prompts[:5])]
    want = LLMEngine(engine_model, num_blocks=256).runner.forward(items)
    monkeypatch.setattr(ModelRunner, "MAX_SEQUENCES", 2)
    got = LLMEngine(engine_model, num_blocks=256).runner.forward(items)
    assert got.shape == want.shape == (7, 1000)
    # products of other row counts may sum in another order
    assert float((got - want).abs().max()) < 0.08 * float(want.abs().max())
