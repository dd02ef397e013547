"""Cases, plain forms and 64-bit definitions of the operators of a shared-prompt serving step:

* ``maps``   - block tables, cache slots and positions of a ragged batch, built from request lengths;
* ``prefix`` - paged attention of a batch whose sequences begin with the same cached prefix;
* ``logits`` - penalties for repeated tokens, token biases and grammar masks on logits.

With ``own`` false the operators run in elementary torch operations; with ``own`` true through the framework's entry
points in ``ajllm_b200.ops.serving``. Sizes come from the repository's model configurations (16 / 8 heads of 128 and
vocabulary 32000 for the 1.3B decoder, 32 / 8 heads of 128 and vocabulary 128256 for the 8B decoder), its serving
benchmark (256 sequences, 8192 new tokens per step) and its context lengths.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 16          # tokens per cache block of the serving engine


def listed() -> list[dict]:
    return [
        # a few interactive users decoding: latency is all that counts
        dict(name="maps decode 8", op="maps", seqs=8, cached_lo=20, cached_hi=900, q_lo=1, q_hi=1, max_blocks=64),
        # the steady state of the serving benchmark: a full batch, one new token each, context up to 4096
        dict(name="maps decode 256", op="maps", seqs=256, cached_lo=128, cached_hi=2560, q_lo=1, q_hi=1, max_blocks=256),
        # one prefill step of the benchmark: ragged prompts on top of partly cached ones, odd lengths
        dict(name="maps prefill 11", op="maps", seqs=11, cached_lo=0, cached_hi=733, q_lo=1, q_hi=1487, max_blocks=139),
        # offline prefill of a large batch of long prompts
        dict(name="maps prefill 64", op="maps", seqs=64, cached_lo=0, cached_hi=4095, q_lo=1024, q_hi=3001, max_blocks=512),
        # a handful of requests behind a short system prompt, 1.3B decoder
        dict(name="prefix decode 4", op="prefix", seqs=4, q_len=1, heads=16, kv_heads=8, head_dim=128, prefix=512,
             suffix_lo=9, suffix_hi=101),
        # chat serving: 64 requests behind a 2k system prompt, 8B decoder
        dict(name="prefix decode 64", op="prefix", seqs=64, q_len=1, heads=32, kv_heads=8, head_dim=128, prefix=2048,
             suffix_lo=16, suffix_hi=512),
        # speculative verification (4 draft tokens) behind a document whose length ends inside a block; 64-wide heads
        dict(name="prefix verify 33x5", op="prefix", seqs=33, q_len=5, heads=32, kv_heads=8, head_dim=64, prefix=4001,
             suffix_lo=5, suffix_hi=301),
        # a full batch asking about one 8k document, the context limit of the 8B decoder
        dict(name="prefix decode 256", op="prefix", seqs=256, q_len=1, heads=32, kv_heads=8, head_dim=128, prefix=7680,
             suffix_lo=32, suffix_hi=512),
        # one request of the 1.3B decoder with penalties
        dict(name="logits 1x32000", op="logits", rows=1, vocab=32000, dtype="bf16", history=257, biases=0, mask=False),
        # constrained decoding of a few requests, everything switched on
        dict(name="logits 16x128256", op="logits", rows=16, vocab=128256, dtype="bf16", history=1024, biases=64, mask=True),
        # odd vocabulary and row count, fp32 logits
        dict(name="logits 77x31999", op="logits", rows=77, vocab=31999, dtype="fp32", history=333, biases=7, mask=True),
        # a full batch of the 8B decoder with long histories
        dict(name="logits 256x128256", op="logits", rows=256, vocab=128256, dtype="bf16", history=2560, biases=16, mask=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """Log-uniform whole number in ``[lo, hi]`` (``lo`` may be 0)."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(max(lo, 0.7)), math.log(hi + 0.999))))))


def draw(rng) -> dict:
    op = rng.choice(["maps", "prefix", "logits"])
    if op == "maps":
        seqs = _log_int(rng, 1, 512)
        q_hi = rng.choice([1, rng.randint(2, 9), _log_int(rng, 10, 4096)])
        q_hi = max(1, min(q_hi, 262144 // (2 * seqs)))
        q_lo = 1 if q_hi < 10 else _log_int(rng, 1, q_hi)
        cached_hi = _log_int(rng, 1, 4095)
        cached_lo = rng.randint(0, cached_hi)
        most = (cached_hi + q_hi + BLOCK - 1) // BLOCK
        return dict(op=op, seqs=seqs, cached_lo=cached_lo, cached_hi=cached_hi, q_lo=q_lo, q_hi=q_hi,
                    max_blocks=most + rng.randint(0, 17))
    if op == "prefix":
        head_dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 8])
        q_len = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 96)])
        prefix = _log_int(rng, 16, 7680)
        suffix_hi = q_len + _log_int(rng, 1, 512)
        suffix_lo = rng.randint(q_len, suffix_hi)
        seqs = _log_int(rng, 2, 256)
        # no more work than the largest listed case
        heads = kv_heads * group
        room = 256 * 32 * 128 * 7680 / (q_len * heads * head_dim * (prefix + suffix_hi))
        seqs = max(1, min(seqs, int(room), 4096 // q_len))
        return dict(op=op, seqs=seqs, q_len=q_len, heads=heads, kv_heads=kv_heads, head_dim=head_dim, prefix=prefix,
                    suffix_lo=suffix_lo, suffix_hi=suffix_hi)
    vocab = rng.choice([32000, 128256, _log_int(rng, 300, 128256)])
    rows = min(_log_int(rng, 1, 512), 256 * 128256 // vocab)
    return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["bf16", "fp32"]), history=_log_int(rng, 0, 2560),
                biases=rng.choice([0, _log_int(rng, 1, 64)]), mask=rng.random() < 0.6)


# --------------------------------------------------------------------------------------------------- inputs


def _spread(lo: int, hi: int, n: int) -> torch.Tensor:
    """``n`` whole numbers spread evenly over ``[lo, hi]``: a case's total work does not depend on the seed, the order
    of the lengths does."""
    return torch.linspace(lo, hi, n, dtype=torch.float64).round().to(torch.int64) if n > 1 else torch.tensor([hi])


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case: dict, seed: int) -> dict:
    return {"maps": _prepare_maps, "prefix": _prepare_prefix, "logits": _prepare_logits}[case["op"]](case, seed)


def _prepare_maps(case: dict, seed: int) -> dict:
    host = torch.Generator().manual_seed(seed)
    n = case["seqs"]
    cached = _spread(case["cached_lo"], case["cached_hi"], n)[torch.randperm(n, generator=host)]
    new = _spread(case["q_lo"], case["q_hi"], n)
    counts = (cached + new + BLOCK - 1) // BLOCK
    blocks = int(counts.sum())
    ids = torch.randperm(2 * blocks + 1, generator=host)[:blocks]
    int32 = dict(dtype=torch.int32, device="cuda")
    total = int(new.sum())
    # the buffers a server keeps from step to step
    kept = (torch.empty(n, case["max_blocks"], **int32), torch.empty(total, **int32),
            torch.empty(total, dtype=torch.int64, device="cuda"), torch.empty(n + 1, **int32), torch.empty(n, **int32))
    return dict(case=case, ids=ids.to(**int32), counts=counts.to(**int32), cached=cached.to(**int32), new=new.to(**int32),
                total=total, kept=kept, pad=2 * blocks + 1)


def _prepare_prefix(case: dict, seed: int) -> dict:
    gen, host = _generator(seed), torch.Generator().manual_seed(seed)
    n, q_len, prefix = case["seqs"], case["q_len"], case["prefix"]
    suffix = _spread(case["suffix_lo"], case["suffix_hi"], n)[torch.randperm(n, generator=host)]
    context = suffix + prefix
    shared = prefix // BLOCK                                    # whole blocks that all sequences have in common
    own_blocks = (context + BLOCK - 1) // BLOCK - shared
    width = shared + int(own_blocks.max())
    order = torch.randperm(shared + int(own_blocks.sum()) + 3, generator=host)
    tables = torch.zeros(n, width, dtype=torch.int64)
    tables[:, :shared] = order[:shared]
    column = torch.arange(width - shared)
    mine = column[None, :] < own_blocks[:, None]
    first = torch.cumsum(own_blocks, 0) - own_blocks
    tables[:, shared:] = torch.where(mine, order[shared + (first[:, None] + column[None, :]).clamp(max=int(own_blocks.sum()) - 1)], 0)
    shape = (order.numel(), BLOCK, case["kv_heads"], case["head_dim"])
    bf16 = dict(dtype=torch.float32, device="cuda", generator=gen)
    keys, values = torch.randn(shape, **bf16).to(torch.bfloat16), torch.randn(shape, **bf16).to(torch.bfloat16)
    tail = prefix - shared * BLOCK
    if tail:
        # the prefix ends inside a block: every sequence holds a copy of its last tokens in its own block
        at = tables[:, shared].cuda()
        keys[at, :tail] = keys[at[0], :tail].clone()
        values[at, :tail] = values[at[0], :tail].clone()
    # queries somewhat longer than unit variance, so that the softmax has peaks
    q = (1.5 * torch.randn(n * q_len, case["heads"], case["head_dim"], **bf16)).to(torch.bfloat16)
    int32 = dict(dtype=torch.int32, device="cuda")
    return dict(case=case, q=q, keys=keys, values=values, tables=tables.to(**int32), context=context.to(**int32),
                suffix_hi=case["suffix_hi"])


def _prepare_logits(case: dict, seed: int) -> dict:
    gen = _generator(seed)
    rows, vocab, longest = case["rows"], case["vocab"], case["history"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    logits = (2.5 * torch.randn(rows, vocab, device="cuda", generator=gen)).to(dtype)
    int32 = dict(dtype=torch.int32, device="cuda")
    lens = _spread(longest // 4, longest, rows).to(**int32)
    prompt = lens // 2
    # word frequencies fall off steeply: many repeats of few tokens
    history = (vocab ** torch.rand(rows, longest, device="cuda", generator=gen) - 1).to(torch.int32).clamp(0, vocab - 1)
    history[torch.arange(longest, device="cuda")[None, :] >= lens[:, None]] = -1
    one = torch.rand(3, rows, device="cuda", generator=gen)
    state = dict(case=case, logits=logits, history=history, prompt=prompt, lens=lens, repetition=1.0 + 0.5 * one[0],
                 presence=one[1] - 0.3, frequency=0.5 * one[2], bias_ids=None, bias_values=None, mask=None)
    if case["biases"]:
        state["bias_ids"] = torch.randint(0, vocab, (rows, case["biases"]), generator=gen, **int32)
        state["bias_values"] = 4 * torch.randn(rows, case["biases"], device="cuda", generator=gen)
    if case["mask"]:
        # a grammar state admits from a few to nearly all tokens: here every word of 32 tokens is shut with its row's share
        words = torch.randint(-2**31, 2**31 - 1, (rows, (vocab + 31) // 32), generator=gen, **int32)
        shut = torch.rand(words.shape, device="cuda", generator=gen) < torch.rand(rows, 1, device="cuda", generator=gen)
        state["mask"] = torch.where(shut, torch.zeros_like(words), words)
    return state


# --------------------------------------------------------------------------------------------------- one pass


def run(state: dict):
    return {"maps": _run_maps, "prefix": _run_prefix, "logits": _run_logits}[state["case"]["op"]](state)


def _run_maps(s: dict):
    case = s["case"]
    if own:
        from ajllm_b200.ops import serving
        return tuple(serving.batch_maps(s["ids"], s["counts"], s["cached"], s["new"], s["total"], case["max_blocks"],
                                        block_size=BLOCK, pad_block=s["pad"], out=s["kept"]))
    n = case["seqs"]
    device = s["ids"].device
    counts, new, cached = s["counts"].long(), s["new"].long(), s["cached"].long()
    first_block = torch.cumsum(counts, 0) - counts
    first_token = torch.cumsum(new, 0) - new
    column = torch.arange(case["max_blocks"], device=device)
    at = (first_block[:, None] + column).clamp(max=s["ids"].numel() - 1)
    tables = torch.where(column < counts[:, None], s["ids"][at], torch.full_like(at, s["pad"], dtype=torch.int32))
    seq = torch.repeat_interleave(torch.arange(n, device=device), new, output_size=s["total"])
    positions = cached[seq] + torch.arange(s["total"], device=device) - first_token[seq]
    block = s["ids"].long()[first_block[seq] + positions // BLOCK]
    slots = block * BLOCK + positions % BLOCK
    q_start = torch.cat((first_token, first_token[-1:] + new[-1:]))
    return tables, positions.int(), slots, q_start.int(), (cached + new).int()


def _prefix_mathematics(s: dict, dtype: torch.dtype) -> torch.Tensor:
    """softmax(q k^T / sqrt(hd)) v: the scores against the shared prefix are one product for the whole batch, those
    against the rest are per sequence; one softmax over both."""
    case = s["case"]
    n, q_len, kv_heads, hd = case["seqs"], case["q_len"], case["kv_heads"], case["head_dim"]
    group = case["heads"] // kv_heads
    shared = case["prefix"] // BLOCK
    whole = shared * BLOCK
    q = s["q"].to(dtype).view(n, q_len, kv_heads, group, hd)
    tables = s["tables"].long()
    pk, pv = (c[tables[0, :shared]].to(dtype).view(whole, kv_heads, hd) for c in (s["keys"], s["values"]))
    rest = tables[:, shared:]
    width = rest.shape[1] * BLOCK
    sk, sv = (c[rest].to(dtype).view(n, width, kv_heads, hd) for c in (s["keys"], s["values"]))
    scores = torch.cat((torch.einsum("nikgd,pkd->nikgp", q, pk), torch.einsum("nikgd,nskd->nikgs", q, sk)), dim=-1) * hd ** -0.5
    last = s["context"].long()[:, None] - q_len + torch.arange(q_len, device=q.device) - whole      # last visible key behind the prefix
    hidden = torch.arange(width, device=q.device) > last[..., None]
    scores[..., whole:].masked_fill_(hidden[:, :, None, None, :], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.einsum("nikgp,pkd->nikgd", p[..., :whole], pv) + torch.einsum("nikgs,nskd->nikgd", p[..., whole:], sv)
    return out.reshape(n * q_len, case["heads"], hd)


def _run_prefix(s: dict):
    if own:
        from ajllm_b200.ops import serving
        return serving.shared_prefix_attention(s["q"], s["keys"], s["values"], s["tables"], s["context"], s["case"]["prefix"],
                                               q_len=s["case"]["q_len"])
    return _prefix_mathematics(s, torch.float32).to(torch.bfloat16)


def _run_logits(s: dict):
    if own:
        from ajllm_b200.ops import serving
        return serving.process_logits(s["logits"], history=s["history"], prompt_lens=s["prompt"], history_lens=s["lens"],
                                      repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                                      bias_ids=s["bias_ids"], bias_values=s["bias_values"], token_mask=s["mask"])
    rows, vocab = s["logits"].shape
    device = s["logits"].device
    x = s["logits"].float()
    place = torch.arange(s["history"].shape[1], device=device)[None, :]
    known = place < s["lens"][:, None]
    made = known & (place >= s["prompt"][:, None])
    ids = s["history"].long().clamp(min=0)
    seen = torch.zeros(rows, vocab, dtype=torch.int32, device=device).scatter_add_(1, ids, known.int())
    count = torch.zeros(rows, vocab, dtype=torch.int32, device=device).scatter_add_(1, ids, made.int())
    factor = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / factor, x * factor), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_ids"] is not None:
        # several biases of one token add up; sums in 64 bits so that their order does not show
        bias = torch.zeros(rows, vocab, dtype=torch.float64, device=device).scatter_add_(1, s["bias_ids"].long(), s["bias_values"].double())
        x = x + bias.float()
    if s["mask"] is not None:
        bit = torch.arange(vocab, device=device)
        x = x.masked_fill((s["mask"][:, bit // 32] >> (bit % 32)) & 1 == 0, float("-inf"))
    return x


# --------------------------------------------------------------------------------------------------- cost and truth


def work(case: dict) -> dict:
    if case["op"] == "maps":
        n = case["seqs"]
        new = _spread(case["q_lo"], case["q_hi"], n)
        # block ids are bounded by the mean context: the order in which lengths meet moves a partial block per sequence at most
        context = int(_spread(case["cached_lo"], case["cached_hi"], n).sum() + new.sum())
        read = 4 * (context // BLOCK + n // 2) + 12 * n
        return {"bytes": read + 4 * n * case["max_blocks"] + 12 * int(new.sum()) + 4 * (2 * n + 1), "flops": 0}
    if case["op"] == "prefix":
        n, q_len, heads, hd = case["seqs"], case["q_len"], case["heads"], case["head_dim"]
        suffix = int(_spread(case["suffix_lo"], case["suffix_hi"], n).sum())
        tokens = case["prefix"] + suffix                                   # the prefix is read once for all
        visible = n * q_len * case["prefix"] + q_len * suffix - n * q_len * (q_len - 1) // 2
        return {"bytes": 2 * 2 * tokens * case["kv_heads"] * hd + 2 * 2 * n * q_len * heads * hd + 4 * (tokens // BLOCK + 2 * n),
                "flops": 4 * visible * heads * hd}
    rows, vocab = case["rows"], case["vocab"]
    lens = int(_spread(case["history"] // 4, case["history"], rows).sum())
    size = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": rows * vocab * (size + 4) + 4 * lens + 8 * rows * case["biases"] + (rows * ((vocab + 31) // 32) * 4 if case["mask"] else 0),
            "flops": rows * vocab}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "maps":
        return None                                  # whole numbers: they are equal or wrong
    if case["op"] == "prefix":
        return _exact_prefix(s)
    return _exact_logits(s)


def _exact_prefix(s: dict) -> torch.Tensor:
    """Every sequence on its own, its whole context laid out in order, in 64 bits."""
    case = s["case"]
    q_len, kv_heads, hd = case["q_len"], case["kv_heads"], case["head_dim"]
    group = case["heads"] // kv_heads
    rows = []
    for i, length in enumerate(s["context"].tolist()):
        blocks = s["tables"][i, :(length + BLOCK - 1) // BLOCK].long()
        k = s["keys"][blocks].reshape(-1, kv_heads, hd)[:length].double().transpose(0, 1)
        v = s["values"][blocks].reshape(-1, kv_heads, hd)[:length].double().transpose(0, 1)
        q = s["q"][i * q_len:(i + 1) * q_len].double().view(q_len, kv_heads, group, hd).permute(1, 2, 0, 3).reshape(kv_heads, group * q_len, hd)
        scores = q @ k.transpose(1, 2) / math.sqrt(hd)
        place = torch.arange(length, device=q.device)
        last = length - q_len + torch.arange(q_len, device=q.device).repeat(group)
        scores = scores.masked_fill(place[None, None, :] > last[None, :, None], -math.inf)
        rows.append((torch.softmax(scores, -1) @ v).view(kv_heads, group, q_len, hd).permute(2, 0, 1, 3).reshape(q_len, case["heads"], hd))
    return torch.cat(rows)


def _exact_logits(s: dict) -> torch.Tensor:
    """Token by token over each row's history, in 64 bits."""
    x = s["logits"].double()
    for r in range(x.shape[0]):
        length, prompt = int(s["lens"][r]), int(s["prompt"][r])
        tokens = s["history"][r, :length].long()
        unique = torch.unique(tokens)
        held = x[r, unique]
        x[r, unique] = torch.where(held > 0, held / s["repetition"][r].double(), held * s["repetition"][r].double())
        made, times = torch.unique(tokens[prompt:], return_counts=True)
        x[r, made] -= s["frequency"][r].double() * times + s["presence"][r].double()
    if s["bias_ids"] is not None:
        x.scatter_add_(1, s["bias_ids"].long(), s["bias_values"].double())
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=x.device)) & 1
        x[bits.flatten(1)[:, :x.shape[1]] == 0] = -math.inf
    return x
