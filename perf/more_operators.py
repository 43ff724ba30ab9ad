"""The 8-bit paged cache and the logits' way to the verification, timed through the public entry points and in plain torch.

``kind`` of a case:
  store    ``store_kvcache_fp8``: a step's keys and values to a cache in e4m3 with a power-of-two scale per block and head
  attend   ``paged_attention_fp8``: causal attention of a decode or verify step, or of a chunk of a prompt, over that cache
  blocks   ``copy_cache_blocks``: blocks of all layers' caches copied (a fork) or moved together (then device tables follow)
  adjust   ``adjust_logits``: penalties for repeated tokens, biases and grammar masks on the rows that are verified next
Heads are those of ``perf/cases.py``, its block size of 256 among smaller ones; vocabularies are generic.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3 = torch.float8_e4m3fn
DEV = "cuda"


def listed():
    return [
        # decode: one new token of 64 sequences, each in the middle of a block of its own
        {"name": "store_decode", "kind": "store", "seqs": 64, "new": 1, "start": 777, "skip": False, "kv_heads": 4, "head_dim": 128, "block": 256, "dtype": "bf16"},
        # prompts: whole blocks, the last one of each sequence in part
        {"name": "store_prompt", "kind": "store", "seqs": 7, "new": 4681, "start": 0, "skip": False, "kv_heads": 8, "head_dim": 128, "block": 256, "dtype": "bf16"},
        # one sequence decoding: latency counts
        {"name": "attend_one", "kind": "attend", "seqs": 1, "q": 1, "low": 777, "high": 777, "empty": False, "heads": 32, "kv_heads": 4, "head_dim": 128, "block": 256, "dtype": "bf16"},
        # a decode batch of mixed lengths
        {"name": "attend_decode", "kind": "attend", "seqs": 64, "q": 1, "low": 750, "high": 3001, "empty": False, "heads": 32, "kv_heads": 4, "head_dim": 128, "block": 256, "dtype": "bf16"},
        # verify of 8 tokens: 64 query rows to a head's keys
        {"name": "attend_verify", "kind": "attend", "seqs": 32, "q": 8, "low": 512, "high": 2048, "empty": False, "heads": 32, "kv_heads": 4, "head_dim": 128, "block": 256, "dtype": "bf16"},
        # small blocks, small heads, a batch with a free place, nothing a multiple of a tile
        {"name": "attend_verify_odd", "kind": "attend", "seqs": 23, "q": 5, "low": 5, "high": 1501, "empty": True, "heads": 14, "kv_heads": 2, "head_dim": 64, "block": 16, "dtype": "fp16"},
        # two long documents, decoding: the cache's bytes bound it
        {"name": "attend_long", "kind": "attend", "seqs": 2, "q": 1, "low": 130001, "high": 131072, "empty": False, "heads": 32, "kv_heads": 8, "head_dim": 128, "block": 256, "dtype": "bf16"},
        # a chunk of a prompt over what is cached of it: the matrix cores bound it
        {"name": "attend_chunk", "kind": "attend", "seqs": 4, "q": 512, "low": 3500, "high": 8192, "empty": False, "heads": 32, "kv_heads": 4, "head_dim": 128, "block": 256, "dtype": "bf16"},
        # eight sequences fork: their last, half-filled blocks are copied in all 48 layers of a 16-bit cache
        {"name": "blocks_fork", "kind": "blocks", "cache": "bf16", "layers": 48, "num_blocks": 96, "pairs": 8, "tables": 0, "kv_heads": 4, "head_dim": 128, "block": 16},
        # an 8-bit cache is compacted: 500 blocks move to free places, and the tables follow
        {"name": "blocks_compact", "kind": "blocks", "cache": "fp8", "layers": 24, "num_blocks": 1100, "pairs": 500, "tables": 64, "kv_heads": 4, "head_dim": 128, "block": 64},
        # a verify batch: penalties over up to 4096 tokens and the drafts, biases, masks on every row
        {"name": "adjust_batch", "kind": "adjust", "seqs": 64, "drafts": 8, "vocab": 131072, "dtype": "bf16", "history": 4096, "bias": 64, "mask": True},
        # one sequence in fp32 with an odd vocabulary and a few drafts: the smallest call
        {"name": "adjust_one_odd", "kind": "adjust", "seqs": 1, "drafts": 4, "vocab": 50257, "dtype": "fp32", "history": 700, "bias": 5, "mask": False},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "blocks", "adjust"])
    kv_heads, group = rng.choice([(4, 8), (8, 4), (2, 7), (16, 1), (1, 8), (4, 7)])
    head_dim, block = rng.choice([64, 128, 128]), rng.choice([16, 32, 48, 64, 128, 256, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "store":
        while True:
            skip = rng.random() < 0.3
            seqs, new = _log_int(rng, 1, 256), rng.randint(2, 9) if skip else rng.choice([1, 1, _log_int(rng, 2, 8192)])
            if seqs * new * kv_heads * head_dim <= 32768 * 1024:
                break
        return {"kind": kind, "seqs": seqs, "new": new, "start": rng.randint(0, 1000) if new < 10 or rng.random() < 0.5 else 0, "skip": skip,
                "kv_heads": kv_heads, "head_dim": head_dim, "block": block, "dtype": dtype}
    if kind == "attend":
        while True:
            seqs, high = _log_int(rng, 1, 256), _log_int(rng, 16, 131072)
            q = min(rng.choice([1, 1, rng.randint(2, 9), rng.randint(2, 9), _log_int(rng, 10, 512)]), high)
            low = rng.randint(q, high)
            keys = seqs * (low + high) / 2 * kv_heads
            if seqs * high * kv_heads * head_dim * 2 <= 537e6 and keys * head_dim * group * q <= 64 * 10 ** 9 and seqs * high * kv_heads * group * q <= 4 * 32 * 512 * 8192:
                break
        return {"kind": kind, "seqs": seqs, "q": q, "low": low, "high": high, "empty": seqs > 1 and rng.random() < 0.3, "heads": kv_heads * group,
                "kv_heads": kv_heads, "head_dim": head_dim, "block": block, "dtype": dtype}
    if kind == "blocks":
        while True:
            layers, pairs, cache = rng.choice([1, 6, 24, 48]), _log_int(rng, 1, 1000), rng.choice(["fp8", "fp8", "bf16"])
            if layers * pairs * block * kv_heads * head_dim * 2 * (1 if cache == "fp8" else 2) <= 24 * 500 * 64 * 4 * 128 * 2:
                break
        return {"kind": kind, "cache": cache, "layers": layers, "num_blocks": 2 * pairs + rng.randint(0, 99), "pairs": pairs,
                "tables": rng.choice([0, rng.randint(1, 200)]), "kv_heads": kv_heads, "head_dim": head_dim, "block": block}
    while True:
        seqs, drafts, vocab = _log_int(rng, 1, 256), rng.choice([0, 1, 3, 5, 8]), _log_int(rng, 1000, 200000)
        if seqs * (drafts + 1) * vocab <= 64 * 8 * 131072:
            break
    return {"kind": kind, "seqs": seqs, "drafts": drafts, "vocab": vocab, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
            "history": _log_int(rng, 1, 16384), "bias": rng.choice([0, 3, 300]), "mask": rng.random() < 0.5}


# ---- inputs -------------------------------------------------------------------------------
def _query_lens(case):
    """Query tokens of each sequence: the first has them all, the others a few less; known to the host."""
    if case["kind"] == "adjust":
        n = case["drafts"] + 1
    else:
        n = case["q"]
    return [n - (7 * s) % (n // 2 + 1) for s in range(case["seqs"])]


def _context_lens(case):
    """Cached tokens of each sequence, the step's own among them; with "empty" one place of the batch is free."""
    lens = [case["low"] + (case["high"] - case["low"]) * s // max(case["seqs"] - 1, 1) for s in range(case["seqs"])]
    if case["empty"]:
        lens[len(lens) // 2] = 0
    return lens


def _starts(lens):
    at, out = 0, []
    for n in lens:
        out.append(at)
        at += n
    return out


def _codes(x, scale):
    return (x / scale[..., None, None]).to(E4M3)


def _scale_of(amax):
    """The smallest power of two (2^-64 at least) that leaves amax / scale within e4m3's largest number, 448."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - torch.where(m > 0.875, 8, 9), -64)
    return torch.ldexp(torch.ones_like(amax), torch.clamp(e, min=-64))


def _filled(randn, blocks, kv_heads, block, head_dim):
    """A cache whose blocks are full of rows that were stored before: codes of K, of V (transposed), and both scales."""
    k, v = randn(blocks, kv_heads, block, head_dim), randn(blocks, kv_heads, head_dim, block)
    scales = torch.stack((_scale_of(k.abs().amax((2, 3))), _scale_of(v.abs().amax((2, 3)))), dim=-1)
    return _codes(k, scales[..., 0]), _codes(v, scales[..., 1]), scales


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    int32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    s = {"case": dict(case)}
    if case["kind"] == "store":
        H, D, bs, dt = case["kv_heads"], case["head_dim"], case["block"], DTYPES[case["dtype"]]
        first = [case["start"] + 13 * i if case["start"] else 0 for i in range(case["seqs"])]
        counts = [(p + case["new"] - 1) // bs - p // bs + 1 for p in first]      # blocks that a sequence's tokens lie in
        places = torch.randperm(sum(counts) + 8, generator=host)
        pos = torch.tensor(first)[:, None] + torch.arange(case["new"])
        which = torch.tensor(_starts(counts))[:, None] + pos // bs - (torch.tensor(first) // bs)[:, None]
        slots = (places[which] * bs + pos % bs).flatten()
        n = slots.numel()
        s["key"], s["value"] = randn(n, H, D).to(dt), randn(n, H, D).to(dt)
        s["src"] = None
        if case["skip"]:                                  # a sequence's first token has its key in the cache
            src = torch.arange(n)
            src = src[src % case["new"] != 0]
            slots, s["src"] = slots[src], src.to(torch.int32).to(DEV)
        s["slots"] = slots.to(torch.int32).to(DEV)
        s["blocks"] = torch.unique(slots // bs).to(DEV)
        s["k"], s["v"], s["scales"] = _filled(randn, places.numel(), H, bs, D)
        return s
    if case["kind"] == "attend":
        H, D, bs, dt = case["kv_heads"], case["head_dim"], case["block"], DTYPES[case["dtype"]]
        q_lens, lens = _query_lens(case), _context_lens(case)
        counts = [(n + bs - 1) // bs for n in lens]
        most = max(max(counts), 1)
        places = torch.randperm(sum(counts) + 8, generator=host).to(torch.int32)
        tables = torch.full((case["seqs"], most), -1, dtype=torch.int32)
        for i, (at, n) in enumerate(zip(_starts(counts), counts)):
            tables[i, :n] = places[at:at + n]
        s["tables"], s["lens"] = tables.to(DEV), int32(lens)
        s["q_lens"], s["longest"] = int32(q_lens), max(q_lens)
        s["q"] = randn(sum(q_lens), case["heads"], D).mul_(1.5).to(dt)
        s["k"], s["v"], s["scales"] = _filled(randn, places.numel(), H, bs, D)
        # where query rows belong, as index tensors for the plain form
        s["row_seq"] = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(q_lens)).to(DEV)
        s["row_at"] = (torch.arange(sum(q_lens)) - torch.tensor(_starts(q_lens)).repeat_interleave(torch.tensor(q_lens))).to(DEV)
        return s
    if case["kind"] == "blocks":
        H, D, bs, nb, L = case["kv_heads"], case["head_dim"], case["block"], case["num_blocks"], case["layers"]
        fill = lambda *shape: torch.randint(-2 ** 31, 2 ** 31, shape[:-1] + (shape[-1] // 4,), generator=g, device=DEV, dtype=torch.int32)  # noqa: E731
        if case["cache"] == "fp8":                        # (no bit pattern is no number)
            codes = lambda *shape: fill(*shape).view(torch.uint8).bitwise_and_(0xBF).view(E4M3)  # noqa: E731
            s["caches"] = [codes(L, nb, H, bs, D), codes(L, nb, H, D, bs),
                           torch.ldexp(torch.ones(L, nb, H, 2, device=DEV), torch.randint(-9, -3, (L, nb, H, 2), generator=g, device=DEV))]
        else:
            rows = lambda: fill(L, nb, bs, 2 * H * D).view(torch.int16).bitwise_and_(-16385).view(torch.bfloat16)  # noqa: E731
            s["caches"] = [rows(), rows()]
        # free places are low, the blocks to be moved high; both lists are the host's, in no order
        low, high = torch.randperm(nb // 2, generator=host), torch.randperm(nb - nb // 2, generator=host)
        s["dst"], s["src"] = low[:case["pairs"]].to(torch.int32), (high[:case["pairs"]] + nb // 2).to(torch.int32)
        s["tables"] = None
        if case["tables"]:
            tables = torch.randint(0, nb, (case["tables"], nb // 4 + 1), generator=host, dtype=torch.int32)
            tables[:, nb // 5:] = -1
            s["tables"] = tables.to(DEV)
        return s
    lens, V, S = _query_lens(case), case["vocab"], case["seqs"]
    n, T = sum(lens), case["history"]
    s["lens"], s["longest"] = int32(lens), max(lens)
    s["logits"] = randn(n, V).mul_(2.5).to(DTYPES[case["dtype"]])
    # words fall off over the ranks as a language's do; a place without history now and then
    word = lambda *shape: (V * torch.rand(*shape, generator=g, device=DEV).pow(4)).long().clamp_(max=V - 1)  # noqa: E731
    s["tokens"], s["drafts"] = word(S, T), word(n - S)
    token_lens = [0 if i % 8 == 5 else T - (T // 2) * i // S for i in range(S)]
    s["token_lens"], s["prompt_lens"] = int32(token_lens), int32([t * (i % 4) // 4 for i, t in enumerate(token_lens)])
    some = lambda *values: torch.tensor(values, device=DEV)[torch.randint(0, len(values), (S,), generator=g, device=DEV)]  # noqa: E731
    s["repetition"], s["frequency"], s["presence"] = some(1.0, 1.1, 1.3), some(0.0, 0.2, 0.5), some(0.0, 0.4)
    s["bias_tokens"] = s["bias_values"] = s["mask"] = None
    if case["bias"]:
        m = case["bias"]
        at = (torch.randint(0, V, (S, 1), generator=g, device=DEV) + torch.arange(m, device=DEV) * (V // m)) % V
        at[:, m - m // 4:] = -1                           # not every sequence has as many
        s["bias_tokens"], s["bias_values"] = at.to(torch.int32), randn(S, m).mul_(4.0)
    if case["mask"]:                                      # bit t % 32 of word t / 32: the grammar allows token t; strict rows and loose ones
        bits = lambda: torch.randint(-2 ** 31, 2 ** 31, (n, (V + 31) // 32), generator=g, device=DEV, dtype=torch.int32)  # noqa: E731
        a, b = bits(), bits()
        strict = (torch.arange(n, device=DEV) % 3 == 0)[:, None]
        s["mask"] = torch.where(strict, a & b & bits() & bits(), a | b)
    seq = torch.repeat_interleave(torch.arange(S), torch.tensor(lens))
    at = torch.arange(n) - torch.tensor(_starts(lens))[seq]
    s["row_seq"] = seq.to(DEV)
    # (row, draft) for every draft that stands before a row of its sequence
    rows = torch.repeat_interleave(torch.arange(n), at)
    before = torch.arange(rows.numel()) - torch.repeat_interleave(torch.cumsum(at, 0) - at, at)
    s["pair_row"], s["pair_draft"] = rows.to(DEV), (torch.tensor(_starts([x - 1 for x in lens]))[seq[rows]] + before).to(DEV)
    return s


# ---- plain forms --------------------------------------------------------------------------
def _plain_rows(x, codes, scales, slots, blocks):
    """Rows x [n, heads, dim] to their slots of codes [blocks, heads, block, dim], a view of the cache, under the blocks' scales."""
    bytes_, bs = codes.view(torch.uint8), codes.shape[2]
    block, at = slots // bs, slots % bs
    amax = torch.zeros_like(scales).scatter_reduce_(0, block[:, None].expand(-1, scales.shape[1]), x.abs().amax(-1), "amax")
    anew = torch.zeros(codes.shape[0], dtype=torch.int32, device=x.device).scatter_reduce_(0, block, (at == 0).int(), "amax")[blocks, None] > 0
    old = torch.where(anew, 0.0, scales[blocks])
    new = torch.maximum(old, _scale_of(amax[blocks]))
    ratio = torch.where(anew, 1.0, old / new)[..., None, None]
    bytes_[blocks] = (bytes_[blocks].view(E4M3).float() * ratio).to(E4M3).view(torch.uint8)
    scales[blocks] = new
    bytes_[block, :, at] = (x / scales[block][..., None]).to(E4M3).view(torch.uint8)


def _plain_store(s):
    key, value, slots = s["key"], s["value"], s["slots"].long()
    if s["src"] is not None:
        key, value = key[s["src"]], value[s["src"]]
    _plain_rows(key.float(), s["k"], s["scales"][..., 0], slots, s["blocks"])
    _plain_rows(value.float(), s["v"].transpose(2, 3), s["scales"][..., 1], slots, s["blocks"])
    return s["k"], s["v"], s["scales"]


def _plain_attend(s):
    case, tables = s["case"], s["tables"].clamp(min=0).long()
    H, D = case["kv_heads"], case["head_dim"]
    G, S, longest = case["heads"] // H, case["seqs"], s["longest"]
    gathered = lambda codes: codes.view(torch.uint8)[tables].view(E4M3).float()  # noqa: E731
    scales = s["scales"][tables][..., None, None]
    k = (gathered(s["k"]) * scales[:, :, :, 0]).permute(0, 2, 1, 3, 4).reshape(S, H, -1, D)
    v = (gathered(s["v"]) * scales[:, :, :, 1]).permute(0, 2, 1, 4, 3).reshape(S, H, -1, D)
    q = torch.zeros(S, longest, H, G, D, device=DEV)
    q[s["row_seq"], s["row_at"]] = s["q"].float().unflatten(1, (H, G))
    x = q.permute(0, 2, 1, 3, 4).reshape(S, H, longest * G, D) @ k.transpose(2, 3) * D ** -0.5
    last = (s["lens"] - s["q_lens"])[:, None] + torch.arange(longest, device=DEV)
    seen = torch.arange(k.shape[2], device=DEV) <= last[:, :, None]
    seen = seen[:, None, :, None].expand(S, 1, longest, G, k.shape[2]).reshape(S, 1, longest * G, -1)
    top = torch.where(seen, x, -math.inf).amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(x - torch.where(top > -math.inf, top, 0.0)), 0.0)
    out = p @ v / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.reshape(S, H, longest, G, D).transpose(1, 2).flatten(2, 3)[s["row_seq"], s["row_at"]].to(s["q"].dtype)


def _plain_blocks(s):
    src, dst = s["src"].to(DEV).long(), s["dst"].to(DEV).long()
    as_bytes = [c.view(torch.uint8) if c.dtype == E4M3 else c for c in s["caches"]]
    as_bytes[0][:, dst], as_bytes[1][:, dst] = as_bytes[0][:, src], as_bytes[1][:, src]
    if len(as_bytes) > 2:
        as_bytes[2][:, dst] = as_bytes[2][:, src]
    if s["tables"] is None:
        return s["caches"]
    names = torch.arange(s["case"]["num_blocks"], dtype=torch.int32, device=DEV)
    names[src] = s["dst"].to(DEV)
    s["tables"].copy_(torch.where(s["tables"] >= 0, names[s["tables"].clamp(min=0).long()], s["tables"]))
    return s["caches"], s["tables"]


def _plain_adjust(s):
    x, seq = s["logits"].float(), s["row_seq"]
    S, V = s["case"]["seqs"], x.shape[1]
    at = torch.arange(s["tokens"].shape[1], device=DEV)
    there, prompt = at < s["token_lens"][:, None], at < s["prompt_lens"][:, None]
    zeros = torch.zeros(S, V, device=DEV)
    seen = zeros.scatter_add(1, s["tokens"], there.float())[seq]
    count = zeros.scatter_add(1, s["tokens"], (there & ~prompt).float())[seq]
    drafted = (s["pair_row"], s["drafts"][s["pair_draft"]])
    one = torch.ones(drafted[0].numel(), device=DEV)
    seen, count = seen.index_put(drafted, one, accumulate=True), count.index_put(drafted, one, accumulate=True)
    r, f, p = (s[name][seq][:, None] for name in ("repetition", "frequency", "presence"))
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - (f * count + p * (count > 0))
    if s["bias_tokens"] is not None:
        to = torch.where(s["bias_tokens"] >= 0, s["bias_tokens"], V).long()
        x = x + torch.zeros(S, V + 1, device=DEV).scatter(1, to, s["bias_values"])[seq, :V]
    if s["mask"] is not None:
        t = torch.arange(V, device=DEV)
        x = torch.where((s["mask"][:, t // 32] >> (t % 32).int()) & 1 == 1, x, -math.inf)
    return x.to(s["logits"].dtype)


# ---- one pass -----------------------------------------------------------------------------
def _own(s):
    import on_device_sd_amd as odsd
    kind = s["case"]["kind"]
    if kind == "store":
        odsd.store_kvcache_fp8(s["key"], s["value"], odsd.KVCacheFP8(s["k"], s["v"], s["scales"]), s["slots"], s["src"])
        return s["k"], s["v"], s["scales"]
    if kind == "attend":
        context = {"block_tables": s["tables"], "context_lens": s["lens"], "max_query_len": s["longest"]}
        if s["longest"] > 1:
            context["verify_query_lens"] = s["q_lens"]
        return odsd.paged_attention_fp8(s["q"], odsd.KVCacheFP8(s["k"], s["v"], s["scales"]), context)
    if kind == "blocks":
        odsd.copy_cache_blocks(s["caches"], s["src"], s["dst"], block_dim=1, block_tables=s["tables"])
        return s["caches"] if s["tables"] is None else (s["caches"], s["tables"])
    context = {"verify_query_lens": s["lens"], "max_query_len": s["longest"]}
    return odsd.adjust_logits(s["logits"], context, tokens=s["tokens"], token_lens=s["token_lens"], prompt_lens=s["prompt_lens"],
                              draft_tokens=s["drafts"], repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                              bias_tokens=s["bias_tokens"], bias_values=s["bias_values"], mask=s["mask"])


def run(s):
    if own:
        return _own(s)
    return {"store": _plain_store, "attend": _plain_attend, "blocks": _plain_blocks, "adjust": _plain_adjust}[s["case"]["kind"]](s)


# ---- what a pass cannot do without ----------------------------------------------------------
def work(case):
    if case["kind"] == "store":
        values = 2 * case["seqs"] * (case["new"] - (1 if case["skip"] else 0)) * case["kv_heads"] * case["head_dim"]
        return {"bytes": values * (SIZES[case["dtype"]] + 1), "flops": 2 * values}
    if case["kind"] == "attend":
        q_lens, lens, e = _query_lens(case), _context_lens(case), SIZES[case["dtype"]]
        pairs = sum(ql * max(n - ql, 0) + ql * (ql + 1) // 2 for ql, n in zip(q_lens, lens) if n)
        return {"bytes": sum(lens) * case["kv_heads"] * case["head_dim"] * 2 + 2 * sum(q_lens) * case["heads"] * case["head_dim"] * e,
                "flops": 4 * pairs * case["heads"] * case["head_dim"]}
    if case["kind"] == "blocks":
        one = 2 * case["kv_heads"] * case["head_dim"] * case["block"] * (1 if case["cache"] == "fp8" else 2) + (8 * case["kv_heads"] if case["cache"] == "fp8" else 0)
        return {"bytes": 2 * case["layers"] * case["pairs"] * one + 4 * case["tables"] * (case["num_blocks"] // 4 + 1), "flops": 0}
    n, V = sum(_query_lens(case)), case["vocab"]
    history = sum(0 if i % 8 == 5 else case["history"] - (case["history"] // 2) * i // case["seqs"] for i in range(case["seqs"]))
    return {"bytes": 2 * n * V * SIZES[case["dtype"]] + 8 * history + (n * ((V + 31) // 32) * 4 if case["mask"] else 0) + 8 * case["seqs"] * case["bias"],
            "flops": 6 * n * V}


# ---- the definitions in 64 bits -------------------------------------------------------------
def _e4m3(y):
    """The nearest of e4m3's numbers, ties to the even one: three bits behind the first, steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -20))), min=-6.0) - 3.0)
    return torch.round(y / step) * step


def _exact_store(s):
    bs, out = s["case"]["block"], []
    slots = s["slots"].cpu().long()
    rows = torch.arange(slots.numel()) if s["src"] is None else s["src"].cpu().long()
    by_block = {}
    for i, slot in enumerate(slots.tolist()):
        by_block.setdefault(slot // bs, []).append((int(rows[i]), slot % bs))
    scales = s["scales"].double()
    for which, (x, codes) in enumerate(((s["key"], s["k"]), (s["value"], s["v"].transpose(2, 3)))):
        held = codes.double()
        for block, pairs in by_block.items():
            at = torch.tensor([p[1] for p in pairs], device=DEV)
            new = x[torch.tensor([p[0] for p in pairs], device=DEV)].double().transpose(0, 1)         # [heads, rows, dim]
            need = new.abs().amax((1, 2)) / 448.0
            need = torch.exp2(torch.ceil(torch.log2(torch.clamp(need, min=2.0 ** -64))))
            if not any(p[1] == 0 for p in pairs):
                old = scales[block, :, which]
                scale = torch.maximum(old, need)
                held[block] = _e4m3(held[block] * (old / scale)[:, None, None])
            else:
                scale = need
            held[block][:, at] = _e4m3(new / scale[:, None, None])
            scales[block, :, which] = scale
        out.append(held if which == 0 else held.transpose(2, 3).contiguous())
    return out[0], out[1], scales


def _exact_attend(s):
    case = s["case"]
    H, D, out = case["kv_heads"], case["head_dim"], []
    G = case["heads"] // H
    first = _starts(_query_lens(case))
    for i, (ql, n) in enumerate(zip(_query_lens(case), _context_lens(case))):
        q = s["q"][first[i]:first[i] + ql].double().reshape(ql, H, G, D)
        o = torch.zeros(ql, H, G, D, dtype=torch.float64, device=DEV)
        blocks = s["tables"][i, :(n + case["block"] - 1) // case["block"]].long()
        for h in range(H if n else 0):
            held = lambda name: s[name][:, h].view(torch.uint8).index_select(0, blocks).view(E4M3).double()  # noqa: E731,B023
            scale = s["scales"][:, h].index_select(0, blocks).double()
            k = (held("k") * scale[:, 0, None, None]).flatten(0, 1)[:n]
            v = (held("v") * scale[:, 1, None, None]).transpose(1, 2).flatten(0, 1)[:n]
            x = torch.mm(q[:, h].flatten(0, 1), k.t()).reshape(ql, G, n).div_(math.sqrt(D))
            hidden = torch.ones(ql, n, dtype=torch.bool, device=DEV).tril_(n - ql).logical_not_()
            o[:, h] = torch.mm(torch.softmax(x.masked_fill_(hidden[:, None], -math.inf), -1).flatten(0, 1), v).reshape(ql, G, D)
        out.append(o.flatten(1, 2))
    return torch.cat(out)


def _exact_blocks(s):
    held = [c.clone() for c in s["caches"]]
    for c, old in zip(held, s["caches"]):
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            c[:, b].copy_(old[:, a])
    if s["tables"] is None:
        return held
    names = dict(zip(s["src"].tolist(), s["dst"].tolist()))
    return held, torch.tensor([[names.get(t, t) for t in row] for row in s["tables"].tolist()], dtype=torch.int32)


def _exact_adjust(s):
    case, V = s["case"], s["case"]["vocab"]
    out, row, draft = [], 0, 0
    token_lens, prompt_lens = s["token_lens"].tolist(), s["prompt_lens"].tolist()
    for i, n in enumerate(_query_lens(case)):
        told = s["tokens"][i, :token_lens[i]]
        r, f, p = (s[name][i].double() for name in ("repetition", "frequency", "presence"))
        bias = torch.zeros(V, dtype=torch.float64, device=DEV)
        if s["bias_tokens"] is not None:
            used = s["bias_tokens"][i] >= 0
            bias[s["bias_tokens"][i][used].long()] = s["bias_values"][i][used].double()
        for j in range(n):
            so_far = torch.cat((told, s["drafts"][draft:draft + j]))
            seen = torch.bincount(so_far, minlength=V) > 0
            count = torch.bincount(so_far[prompt_lens[i]:], minlength=V)
            x = s["logits"][row + j].double()
            x = torch.where(seen & (x > 0), x / r, torch.where(seen, x * r, x)) - f * count - p * (count > 0) + bias
            if s["mask"] is not None:
                allowed = (s["mask"][row + j][:, None] >> torch.arange(32, device=DEV, dtype=torch.int32)).bitwise_and(1).flatten()[:V]
                x = x.masked_fill(allowed == 0, -math.inf)
            out.append(x.to(torch.float64))
        row, draft = row + n, draft + n - 1
    return torch.stack(out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "blocks": _exact_blocks, "adjust": _exact_adjust}[case["kind"]](s)
