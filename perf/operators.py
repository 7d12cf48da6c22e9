"""The operators of branching decode, in plain torch and through the framework: what a benchmark of them runs.

Five operators: the log probabilities of a batch of logits rows (given token, rank, entropy, top
alternatives), and the pages of a paged KV cache copied, forked, freed and compacted.  ``run`` computes
them with elementary torch operations, or, where ``own`` is true, through ``nebulasd_b200``.

Layouts are the framework's: caches ``[num_blocks, num_layers, num_kv_heads, 16, 128]`` fp16, block
table ``[rows, max_blocks]`` int32 with -1 in unused entries, one reference count per block (0: free).
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
BLOCK = 16    # tokens per block
DIM = 128     # head dim
VOCAB = 151936
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One decoding request that asked for its alternatives: the smallest call.
        dict(name="logprobs_one_row", op="logprobs", rows=1, vocab=VOCAB, pad=0, dtype="float16", num_top=20,
             banned=0.0, spread=2.5),
        # The verify rows of 16 requests at depth 4, five alternatives each.
        dict(name="logprobs_verify_16x5", op="logprobs", rows=80, vocab=VOCAB, pad=0, dtype="float16", num_top=5,
             banned=0.0, spread=2.5),
        # A 2,048-token prompt scored token by token.
        dict(name="logprobs_prompt_2048", op="logprobs", rows=2048, vocab=VOCAB, pad=0, dtype="float16", num_top=5,
             banned=0.0, spread=2.5),
        # Grammar-constrained rows in fp32: most tokens banned (-inf), an odd vocabulary in a wider buffer.
        dict(name="logprobs_masked_f32", op="logprobs", rows=333, vocab=50021, pad=11, dtype="float32", num_top=20,
             banned=0.97, spread=4.0),
        # Partial blocks of 64 draft beams (28 layers).
        dict(name="copy_partial_0p6b", op="copy", pairs=64, partial=True, layers=28, kv_heads=8, pool=1024),
        # Whole blocks moved within the 36-layer pool.
        dict(name="copy_full_8b", op="copy", pairs=512, partial=False, layers=36, kv_heads=8, pool=2048),
        # Three more beams for each of 16 requests, 64 tokens of room each (36 layers).
        dict(name="fork_beams_8b", op="fork", requests=16, fan=1, children=48, ctx_lo=256, ctx_hi=4096, room=64,
             layers=36, kv_heads=8, pool=4096),
        # Long prefixes branched once each: tables and reference counts, a one-layer cache.
        dict(name="fork_long", op="fork", requests=64, fan=1, children=64, ctx_lo=8192, ctx_hi=32768, room=0,
             layers=1, kv_heads=8, pool=132 * 1024),
        # The losing beams of 16 requests dropped.
        dict(name="free_beams", op="free", requests=16, fan=4, drop=48, ctx_lo=256, ctx_hi=4096, layers=1,
             kv_heads=1, pool=4096),
        # Most of a batch of long requests ended.
        dict(name="free_long", op="free", requests=64, fan=1, drop=56, ctx_lo=8192, ctx_hi=32768, layers=1,
             kv_heads=1, pool=132 * 1024),
        # Half-empty draft pool.
        dict(name="compact_0p6b", op="compact", requests=4, fan=2, ctx_lo=256, ctx_hi=2048, layers=28, kv_heads=8,
             pool=512),
        # The 36-layer pool with about half of its blocks live, scattered.
        dict(name="compact_8b", op="compact", requests=15, fan=2, ctx_lo=256, ctx_hi=4096, layers=36, kv_heads=8,
             pool=4096),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "copy", "fork", "free", "compact"])
    if op == "logprobs":
        dtype = rng.choice(["float16", "bfloat16", "float32"])
        vocab = _log(rng, 97, VOCAB)
        most = 2048 * VOCAB // vocab // (2 if dtype == "float32" else 1)
        return dict(op=op, rows=_log(rng, 1, min(2048, most)), vocab=vocab, pad=rng.choice([0, 0, 1, 7, 64]),
                    dtype=dtype, num_top=rng.choice([0, 1, 2, 5, 20, 32]), banned=rng.choice([0.0, 0.0, 0.5, 0.99]),
                    spread=rng.uniform(0.5, 6.0))
    layers, kv_heads = _log(rng, 1, 36), rng.choice([1, 2, 4, 8])
    if op == "copy":
        pool = _log(rng, 64, 2048)
        return dict(op=op, pairs=_log(rng, 1, pool // 4), partial=rng.random() < 0.5, layers=layers,
                    kv_heads=kv_heads, pool=pool)
    requests, fan = _log(rng, 1, 16), rng.choice([1, 2, 4])
    lo = _log(rng, 1, 512)
    hi = _log(rng, lo, 4096 // fan)
    case = dict(op=op, requests=requests, fan=fan, ctx_lo=lo, ctx_hi=hi, layers=layers, kv_heads=kv_heads)
    need = max(2, requests) * (hi // BLOCK + 1 + fan)
    if op == "fork":
        case["children"], case["room"] = _log(rng, 1, 64), rng.choice([0, 5, 64])
        need += case["children"] * (2 + case["room"] // BLOCK)
    elif op == "free":
        case["requests"] = requests = max(2, requests)
        case["drop"] = rng.randint(1, requests * fan - 1)
        case["layers"] = case["kv_heads"] = 1
    case["pool"] = min(4096, need + _log(rng, 1, 4096)) if need <= 4096 else need
    return case


# ------------------------------------------------------------------ inputs
def _caches(case, gen):
    shape = (case["pool"], case["layers"], case["kv_heads"], BLOCK, DIM)
    return tuple(torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float16) for _ in range(2))


def _pool(case, rng, gen, extra_rows):
    """A pool in use: `requests` sequences of `fan` rows each that share all blocks but the last, in blocks drawn
    at random, `extra_rows` empty rows, the rows in random order.  The three tables lie in one buffer, so that
    a pass can start from the same pool again with one copy."""
    ctx = rng.integers(case["ctx_lo"], case["ctx_hi"] + 1, size=case["requests"])
    fan, pool = case["fan"], case["pool"]
    rows = case["requests"] * fan + extra_rows
    wide = (case["ctx_hi"] + case.get("room", 0)) // BLOCK + 2
    table, count, length = np.full((rows, wide), -1, np.int32), np.zeros(rows, np.int32), np.zeros(rows, np.int64)
    order, blocks, used = rng.permutation(rows), rng.permutation(pool).astype(np.int32), 0
    for i, c in enumerate(ctx.tolist()):
        n = -(-c // BLOCK)
        if used + n - 1 + fan > pool:
            raise ValueError("the pool is too small")
        shared = blocks[used:used + n - 1]
        for f in range(fan):
            r = order[i * fan + f]
            table[r, :n - 1] = shared
            table[r, n - 1] = blocks[used + n - 1 + f]
            count[r], length[r] = n, c
        used += n - 1 + fan
    refs = np.bincount(table[table >= 0], minlength=pool).astype(np.int32)
    up = lambda n: -(-n // 64) * 64  # noqa: E731
    flat = np.zeros(up(table.size) + up(rows) + pool, np.int32)
    flat[:table.size] = table.reshape(-1)
    flat[up(table.size):up(table.size) + rows] = count
    flat[up(table.size) + up(rows):] = refs
    kept = torch.from_numpy(flat).to(DEVICE)
    meta = kept.clone()
    k, v = _caches(case, gen)
    live = order[:case["requests"] * fan]
    return dict(op=case["op"], k=k, v=v, kept=kept, meta=meta, table=meta[:table.size].view(rows, wide),
                seq_blocks=meta[up(table.size):up(table.size) + rows], refs=meta[up(table.size) + up(rows):],
                ), live, order[case["requests"] * fan:], length


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    op = case["op"]
    if op == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        wide = torch.randn((rows, vocab + case["pad"]), generator=gen, device=DEVICE, dtype=torch.float32)
        x = wide[:, :vocab]
        x *= case["spread"]
        # Model logits: each row has a few tokens that stand out, by anything from nothing to certainty.
        n = min(4, vocab)
        picks = torch.randint(0, vocab, (rows, n), generator=gen, device=DEVICE)
        x.scatter_add_(1, picks, 14 * torch.rand((rows, n), generator=gen, device=DEVICE))
        if case["banned"]:
            ban = torch.rand(vocab, generator=gen, device=DEVICE) < case["banned"]
            ban[0] = False
            x[:, ban] = -math.inf
        # Half of the given tokens are ones the model prefers, half are any.
        other = torch.randint(0, vocab, (rows,), generator=gen, device=DEVICE)
        tokens = torch.where(torch.rand(rows, generator=gen, device=DEVICE) < 0.5, x.argmax(1), other)
        return dict(op=op, logits=wide.to(DTYPES[case["dtype"]])[:, :vocab], tokens=tokens.to(torch.int32),
                    num_top=min(case["num_top"], vocab))
    if op == "copy":
        k, v = _caches(case, gen)
        perm = rng.permutation(case["pool"])[:2 * case["pairs"]]
        tokens = _ints(rng.integers(1, BLOCK + 1, size=case["pairs"])) if case["partial"] else None
        return dict(op=op, k=k, v=v, src=_ints(perm[::2]), dst=_ints(perm[1::2]), tokens=tokens)
    state, live, empty, length = _pool(case, rng, gen, case.get("children", 0))
    if op == "fork":
        parents = rng.choice(live, size=case["children"])
        state.update(parents=_ints(parents), children=_ints(empty), lens=_ints(length[parents]),
                     room=_ints(length[parents] + case["room"]))
    elif op == "free":
        state.update(rows=_ints(rng.permutation(live)[:case["drop"]]))
    return state


# ------------------------------------------------------------------ plain forms
def _ordered(x):
    """int64 keys that order fp32 values as the operators do: by value, -0 as +0, ties to the lowest index."""
    bits = (x + 0.0).view(torch.int32)
    bits = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)
    at = torch.arange(x.shape[1], device=x.device)
    return (bits << 32) | (0xFFFFFFFF - at)


def _plain_logprobs(s):
    x = s["logits"].to(torch.float32)
    t = s["tokens"].to(torch.int64)[:, None]
    top = x.max(1, keepdim=True).values
    d = x - top
    e = d.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    given = x.gather(1, t)
    entropy = log_total - (e * d.clamp(min=-200.0)).sum(1, keepdim=True) / total
    out = dict(logprobs=((given - top) - log_total)[:, 0], ranks=(1 + (x > given).sum(1)).to(torch.int32),
               entropy=entropy[:, 0])
    if s["num_top"]:
        key = _ordered(x).topk(s["num_top"], 1).values
        ids = 0xFFFFFFFF - (key & 0xFFFFFFFF)
        out["top_ids"] = ids.to(torch.int32)
        out["top_logprobs"] = (x.gather(1, ids) - top) - log_total
    return out


def _plain_copy(k, v, src, dst, tokens):
    src, dst = src.long(), dst.long()
    if tokens is None:
        k[dst], v[dst] = k[src], v[src]
        return
    live = (torch.arange(BLOCK, device=k.device) < tokens[:, None])[:, None, None, :, None]
    k[dst] = torch.where(live, k[src], k[dst])
    v[dst] = torch.where(live, v[src], v[dst])


def _plain_fork(s):
    table, refs, pool = s["table"], s["refs"], s["refs"].numel()
    parents, children, lens = s["parents"].long(), s["children"].long(), s["lens"].long()
    shared = lens // BLOCK
    total = (torch.maximum(lens, s["room"].long()) + BLOCK - 1) // BLOCK
    need = total - shared
    end = need.cumsum(0)
    free = refs == 0
    slot = (free.cumsum(0) - 1)
    granted = (end <= free.sum()) | (need == 0)
    by_rank = torch.zeros(pool + 1, dtype=torch.int64, device=table.device)
    by_rank[torch.where(free, slot, pool)] = torch.arange(pool, device=table.device)
    col = torch.arange(table.shape[1], device=table.device)
    parent_rows = table[parents].long()
    fresh = by_rank[((end - need)[:, None] + col - shared[:, None]).clamp(0, pool - 1)]
    is_shared = (col < shared[:, None]) & granted[:, None]
    is_fresh = (col >= shared[:, None]) & (col < total[:, None]) & granted[:, None]
    rows = torch.where(is_shared, parent_rows, torch.where(is_fresh, fresh, table[children].long()))
    refs.index_add_(0, rows.clamp(min=0).reshape(-1), (is_shared | is_fresh).reshape(-1).to(torch.int32))
    table[children] = rows.to(torch.int32)
    s["seq_blocks"][children] = torch.where(granted, total, s["seq_blocks"][children].long()).to(torch.int32)
    part = (granted & (lens % BLOCK > 0)).nonzero()[:, 0]
    at = shared[part][:, None]
    _plain_copy(s["k"], s["v"], parent_rows[part].gather(1, at)[:, 0], rows[part].gather(1, at)[:, 0],
                (lens % BLOCK)[part])


def _plain_free(s):
    table, rows = s["table"], s["rows"].long()
    held = torch.arange(table.shape[1], device=table.device) < s["seq_blocks"][rows][:, None]
    ids = table[rows]
    s["refs"].index_add_(0, ids.clamp(min=0).reshape(-1).long(), -held.reshape(-1).to(torch.int32))
    table[rows] = torch.where(held, -1, ids)
    s["seq_blocks"][rows] = 0


def _plain_compact(s):
    table, refs = s["table"], s["refs"]
    live = refs > 0
    at = torch.arange(refs.numel(), device=refs.device)
    low = at < live.sum()
    dst, src = (~live & low).nonzero()[:, 0], (live & ~low).nonzero()[:, 0]
    moved = torch.where(live, at, -1).to(torch.int32)
    moved[src] = dst.to(torch.int32)
    _plain_copy(s["k"], s["v"], src, dst, None)
    refs[dst] = refs[src]
    refs[src] = 0
    held = torch.arange(table.shape[1], device=table.device) < s["seq_blocks"][:, None]
    table.copy_(torch.where(held, moved[table.clamp(min=0).long()], table))
    return moved


# ------------------------------------------------------------------ the framework's calls
def _own_logprobs(s):
    from nebulasd_b200.logprobs import token_logprobs
    got = token_logprobs(s["logits"], s["tokens"], s["num_top"])
    out = dict(logprobs=got.logprobs, ranks=got.ranks, entropy=got.entropy)
    if s["num_top"]:
        out.update(top_ids=got.top_ids, top_logprobs=got.top_logprobs)
    return out


def _handle(s):
    """The pool's handle, which a program makes once for its tensors and keeps."""
    if "handle" not in s:
        from nebulasd_b200.block_pool import BlockPool
        s["handle"] = BlockPool(s["k"], s["v"], s["table"], s["seq_blocks"], s["refs"])
    return s["handle"]


def _own_copy(s):
    from nebulasd_b200.block_pool import copy_blocks
    copy_blocks(s["k"], s["v"], s["src"], s["dst"], s["tokens"])


def run(state):
    s, op = state, state["op"]
    if op == "logprobs":
        return _own_logprobs(s) if own else _plain_logprobs(s)
    # Caches as the 16-bit words that were copied.
    words = dict(k=s["k"].view(torch.int16), v=s["v"].view(torch.int16))
    if op == "copy":
        if own:
            _own_copy(s)
        else:
            _plain_copy(s["k"], s["v"], s["src"], s["dst"], s["tokens"])
        return words
    # Every pass meets the same pool: its tables are put back first, by the same copy on both sides.
    s["meta"].copy_(s["kept"])
    tables = dict(table=s["table"], seq_blocks=s["seq_blocks"], refs=s["refs"])
    if op == "fork":
        if own:
            _handle(s).fork(s["parents"], s["children"], s["lens"], s["room"])
        else:
            _plain_fork(s)
        return {**tables, **words}
    if op == "free":
        if own:
            _handle(s).free(s["rows"])
        else:
            _plain_free(s)
        return tables
    return {**tables, **words, "moved": _handle(s).compact() if own else _plain_compact(s)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "logprobs":
        n, size = case["rows"] * case["vocab"], DTYPES[case["dtype"]].itemsize
        # per logit: difference, exp, two sums, two comparisons
        return {"bytes": n * size + case["rows"] * (16 + 8 * case["num_top"]), "flops": 6 * n}
    token = 2 * case["layers"] * case["kv_heads"] * DIM * 2  # K and V bytes of one token
    if op == "copy":
        tokens = case["pairs"] * ((BLOCK + 1) / 2 if case["partial"] else BLOCK)
        return {"bytes": 2 * tokens * token + 8 * case["pairs"], "flops": 0}
    ctx = (case["ctx_lo"] + case["ctx_hi"]) / 2
    blocks = ctx / BLOCK + 0.5
    if op == "fork":
        entries = case["children"] * (blocks + case["room"] / BLOCK)
        # entries read, written and counted (read and written), the free blocks looked for, the partial blocks copied
        return {"bytes": 16 * entries + 4 * case["pool"] + case["children"] * (BLOCK - 1) * token, "flops": 0}
    if op == "free":
        return {"bytes": 16 * case["drop"] * blocks, "flops": 0}
    live = min(case["pool"], case["requests"] * (blocks - 1 + case["fan"]))
    moved = live * (1 - live / case["pool"])
    return {"bytes": 2 * moved * BLOCK * token + 8 * case["requests"] * case["fan"] * blocks + 12 * case["pool"],
            "flops": 0}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    """Log probabilities only: what the page operators return is moved or whole, never computed."""
    if case["op"] != "logprobs":
        return None
    s = prepare(case, seed)
    parts = []
    step = max(1, (1 << 27) // case["vocab"])
    for r in range(0, case["rows"], step):
        x, t = s["logits"][r:r + step].double(), s["tokens"][r:r + step].long()
        logp = torch.log_softmax(x, 1)
        p = logp.exp()
        part = [logp[torch.arange(len(t), device=t.device), t],
                (x > x[torch.arange(len(t), device=t.device), t][:, None]).sum(1).int() + 1,
                -torch.where(p > 0, p * logp, 0.0).sum(1)]
        if s["num_top"]:
            ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["num_top"]]
            part += [ids.int(), logp.gather(1, ids)]
        parts.append(part)
    names = ["logprobs", "ranks", "entropy", "top_ids", "top_logprobs"]
    return {n: torch.cat(v) for n, v in zip(names, zip(*parts))}
