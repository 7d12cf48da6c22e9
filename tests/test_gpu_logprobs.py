"""GPU: log probabilities, ranks, entropy and top alternatives against their definitions in 64 bits.

Tolerance: sums are fp32 over at most ``ceil(vocab / 128)`` terms of one thread, joined in a tree; each
term and each addition is off by a few units of 2^-24, so ``s`` and ``w`` are off by at most
``g = (ceil(vocab / 128) + 64) * 2^-24`` of their size.  ``log p = (x - m) - ln s`` is then off by ``g``
plus the rounding of its parts, the entropy ``ln s - w / s`` by ``g (1 + 2 |entropy|)`` likewise; both lie
within ``4 g (1 + |reference|)``.
"""
import math

import pytest
import torch

from oracle.logprobs import token_logprobs as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _close(got, want, vocab):
    got, want = got.double().cpu(), torch.as_tensor(want)
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fin = torch.isfinite(want)
    assert bool(torch.isfinite(got[fin]).all())
    g = (-(-vocab // 128) + 64) * 2.0 ** -24
    err = (got[fin] - want[fin]).abs() - 4 * g * (1 + want[fin].abs())
    assert err.numel() == 0 or float(err.max()) <= 0


def _check(logits, tokens, num_top):
    from nebulasd_b200.logprobs import token_logprobs
    got = token_logprobs(logits, tokens, num_top)
    lp, rk, ent, ids, tops = oracle(logits, None if tokens is None else tokens.tolist(), num_top)
    vocab = logits.shape[1]
    _close(got.entropy, ent, vocab)
    if tokens is None:
        assert got.logprobs is None and got.ranks is None
    else:
        _close(got.logprobs, lp, vocab)
        assert got.ranks.tolist() == rk.tolist()
    if num_top:
        assert got.top_ids.tolist() == ids.tolist()
        _close(got.top_logprobs, tops, vocab)
    else:
        assert got.top_ids is None and got.top_logprobs is None
    return got


def _logits(seed, rows, vocab, dtype, dev, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g) * spread
    x[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] += 12 * torch.rand(rows, generator=g)
    return x.to(dtype).to(dev), torch.randint(0, vocab, (rows,), generator=g).to(torch.int32).to(dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,num_top", [
    (1, 151936, 20), (1, 1, 1), (3, 2, 2), (2, 31, 31), (5, 32, 32), (2, 257, 5), (7, 8191, 32), (4, 8192, 1),
    (4, 8193, 3), (3, 16391, 20), (80, 2048, 0), (9, 32000, 32), (33, 50021, 7), (150, 4099, 5), (700, 1003, 2),
])
def test_matches_the_definition(dtype, rows, vocab, num_top, cuda):
    logits, tokens = _logits(rows + vocab, rows, vocab, dtype, cuda)
    _check(logits, tokens, num_top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,width", [(0, 50048), (3, 50021), (1, 40001), (7, 20011)])
def test_rows_that_start_anywhere(dtype, offset, width, cuda):
    wide, tokens = _logits(offset, 6, 50051, dtype, cuda)
    logits = wide[:, offset:offset + width]
    _check(logits, tokens % width, 9)
    _check(wide[1::2, offset:offset + width], tokens[:3] % width, 9)   # every second row
    _check(wide[:1].expand(4, -1)[:, offset:offset + width], tokens[:4] % width, 2)  # one row, stride 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_optional(dtype, cuda):
    logits, tokens = _logits(5, 11, 9973, dtype, cuda)
    _check(logits, None, 0)
    _check(logits, None, 4)
    tokens[3] = -1
    got = _check(logits, tokens, 4)
    assert math.isnan(float(got.logprobs[3])) and int(got.ranks[3]) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_and_order(dtype, cuda):
    vocab = 40000
    logits = torch.full((8, vocab), -1.0)
    logits[0, [39999, 7, 20000, 123]] = 3.0                 # ties: lowest index first
    logits[1] = 0.0
    logits[1, ::3] = -0.0                                    # signed zeros are one value
    logits[2] = torch.arange(vocab) % 128                    # every value many times
    logits[3] = torch.arange(vocab).flip(0) / vocab          # falling
    logits[4] = torch.arange(vocab) / vocab                  # rising: each tile beats the last
    logits[5] = 2.0                                          # constant
    logits[6, -1] = 1.0                                      # the last
    logits[7] = torch.linspace(-60000, 60000, vocab)[torch.randperm(vocab, generator=torch.Generator().manual_seed(1))]
    tokens = torch.tensor([123, 1, 500, 39999, 0, 39999, 39999, 77], dtype=torch.int32, device=cuda)
    for k in (1, 5, 32):
        _check(logits.to(dtype).to(cuda), tokens, k)


@pytest.mark.parametrize("rows", [3, 500])
@pytest.mark.parametrize("num_top", [1, 8, 9, 32])
def test_lists_that_run_over(rows, num_top, cuda):
    """Rising logits in every warp's range: candidates without end while other warps list and raise the threshold."""
    vocab = 40009
    at = torch.arange(vocab)
    x = torch.stack([(at * (1 + r % 3) + 17 * r) % 4096 / 256.0 if r % 2 else at / vocab for r in range(rows)])
    tokens = torch.arange(rows, dtype=torch.int32) * 79 % vocab
    _check(x.float().to(cuda), tokens.to(cuda), num_top)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masks(dtype, cuda):
    vocab, inf = 20011, math.inf
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(3)
    base = torch.randn((12, vocab), generator=g) * 2
    base[0, 5:] = -inf                     # five tokens left
    base[1, :] = -inf
    base[1, 19000] = 0.5                   # one left
    base[2, :] = -inf                      # none left
    base[3, 100:] = low                    # masked by the type's lowest value
    base[4, :] = low                       # all at the lowest value: uniform
    base[5, :] = -inf
    base[5, 7:9] = low                     # two at the lowest value, the rest banned
    base[6, 11] = math.nan
    base[7, 11] = inf
    base[8, [3, 4]] = math.nan
    base[8, 5] = inf
    base[9, :15000] = -inf                 # whole tiles banned
    base[10, :] = torch.finfo(dtype).max   # all at the highest
    base[11, 3] = torch.finfo(dtype).max
    base[9, [100, 14000]] = low            # (and two masked otherwise)
    tokens = torch.tensor([2, 19000, 4, 200, 9, 7, 11, 11, 4, 14, 3, 4], dtype=torch.int32, device=cuda)
    for k in (0, 6, 32):
        got = _check(base.to(dtype).to(cuda), tokens, k)
    assert got.top_ids[2].tolist() == list(range(32))
    assert abs(float(got.entropy[4]) - math.log(vocab)) < 1e-3
    assert abs(float(got.entropy[5]) - math.log(2)) < 1e-6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 40, 500])
def test_confident_rows_keep_their_precision(dtype, rows, cuda):
    """log p = -log1p(r) of a nearly certain token, to the relative precision of r (``g`` as above)."""
    from nebulasd_b200.logprobs import token_logprobs
    vocab = 20000
    logits, tokens = _logits(rows, rows, vocab, dtype, cuda, spread=1.0)
    logits[torch.arange(rows), tokens.long()] = torch.linspace(12, 24, rows, device=cuda).to(dtype)
    got = token_logprobs(logits, tokens, 1)
    lp, rk, ent, ids, tops = oracle(logits, tokens.tolist(), 1)
    g = (-(-vocab // 128) + 64) * 2.0 ** -24
    for a, b in ((got.logprobs, lp), (got.entropy, ent), (got.top_logprobs, tops)):
        a, b = a.double().cpu(), torch.as_tensor(b)
        assert bool(((a - b).abs() <= 4 * g * b.abs()).all())
    assert got.ranks.tolist() == rk.tolist() and got.top_ids.tolist() == ids.tolist()


@pytest.mark.parametrize("dtype,top,rest", [(torch.float16, -65024.0, -65056.0), (torch.float32, 70000.0, 69980.0),
                                            (torch.float32, -70000.0, -70024.0), (torch.float32, 1e6, 1e6 - 15.0)])
@pytest.mark.parametrize("rows", [1, 500])
def test_confident_rows_far_from_zero_keep_their_precision(dtype, top, rest, rows, cuda):
    """The same where the logits are too far from 0 for the one-pass sums."""
    from nebulasd_b200.logprobs import token_logprobs
    vocab = 20000
    _, tokens = _logits(rows, rows, vocab, dtype, cuda)
    logits = torch.full((rows, vocab), rest, dtype=dtype, device=cuda)
    logits[:, ::5] = -math.inf
    logits[torch.arange(rows), tokens.long()] = top
    logits[0, ::2] = top  # (one with many at the maximum)
    got = token_logprobs(logits, tokens, 2)
    lp, rk, ent, ids, tops = oracle(logits, tokens.tolist(), 2)
    g = (-(-vocab // 128) + 64) * 2.0 ** -24
    for a, b in ((got.logprobs, lp), (got.entropy, ent), (got.top_logprobs, tops)):
        a, b = a.double().cpu(), torch.as_tensor(b)
        assert bool(((a - b).abs() <= 4 * g * b.abs()).all())
    assert got.ranks.tolist() == rk.tolist() and got.top_ids.tolist() == ids.tolist()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 30, 500])
def test_fewer_allowed_tokens_than_alternatives(dtype, rows, cuda):
    """A grammar's mask: a few tokens left, some ruled out by the lowest value, the others by -inf."""
    vocab = 12345
    g = torch.Generator().manual_seed(rows)
    x = torch.full((rows, vocab), -math.inf)
    for r in range(rows):
        at = torch.randperm(vocab, generator=g)
        x[r, at[:r % 9]] = torch.randn(r % 9, generator=g)
        x[r, at[10:10 + r % 5]] = torch.finfo(dtype).min
        if r % 3 == 0:
            x[r, at[20:40]] = -66000.0 if dtype != torch.float16 else -65250.0
    _check(x.to(dtype).to(cuda), torch.randint(0, vocab, (rows,), generator=g).to(torch.int32).to(cuda), 20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,offset", [(1, 0), (9, 3), (480, 5)])
def test_rows_without_a_finite_share(dtype, rows, offset, cuda):
    """Rows with a NaN or +inf and wholly masked ones among others, by one CTA and by several."""
    vocab = 12007
    x, tokens = _logits(rows, rows, vocab + offset, dtype, "cpu")
    tokens = (tokens % vocab).to(cuda)
    low = torch.finfo(dtype).min
    for i in range(0, rows, 3):
        kind = (i // 3) % 5
        if kind == 0:
            x[i] = low
            x[i, ::7] = -math.inf
        elif kind == 1:
            x[i, 5 + 11 * i::400] = math.nan
        elif kind == 2:
            x[i, -1] = math.inf
        elif kind == 3:
            x[i] = math.nan
        else:
            x[i] = -70000. - torch.arange(vocab + offset) if dtype != torch.float16 else low
    for k in (1, 20, 32):
        _check(x.to(cuda)[:, offset:], tokens, k)


def test_row_splits_give_one_answer(cuda):
    """A row's ids and rank do not depend on how many rows are scored with it, its sums only in rounding."""
    from nebulasd_b200.logprobs import token_logprobs
    logits, tokens = _logits(8, 600, 30011, torch.float16, cuda)
    whole = token_logprobs(logits, tokens, 8)
    for rows in (1, 4, 20, 80, 300):
        part = token_logprobs(logits[:rows], tokens[:rows], 8)
        assert torch.equal(part.top_ids, whole.top_ids[:rows]) and torch.equal(part.ranks, whole.ranks[:rows])
        _close(part.entropy, whole.entropy[:rows].double().cpu(), 30011)
        _close(part.logprobs, whole.logprobs[:rows].double().cpu(), 30011)
    again = token_logprobs(logits, tokens, 8)
    assert all(torch.equal(a, b) for a, b in zip(again, whole))  # bit for bit


def test_many_rows_and_far_offsets(cuda):
    """Row offsets beyond 2^31 elements."""
    rows, stride = 5, 600_000_000
    store = torch.empty(4 * stride + 1000, dtype=torch.float16, device=cuda)
    logits = store.as_strided((rows, 1000), (stride, 1))
    x, tokens = _logits(2, rows, 1000, torch.float16, cuda)
    logits.copy_(x)
    _check(logits, tokens, 5)


def test_invalid_tokens_are_reported(cuda):
    from nebulasd_b200.logprobs import token_logprobs, workspace_errors
    logits, tokens = _logits(4, 4, 100, torch.float16, cuda)
    workspace_errors()
    token_logprobs(logits, tokens, 0)
    assert workspace_errors() == 0
    bad = torch.tensor([3, 100, -2, 2 ** 31 - 1], dtype=torch.int32, device=cuda)
    got = token_logprobs(logits, bad, 2)
    assert workspace_errors() == 64 and workspace_errors() == 0
    assert got.ranks.tolist()[1:] == [0, 0, 0] and torch.isnan(got.logprobs[1:]).all()
    assert torch.isfinite(got.entropy).all()


def test_streams_and_graphs(cuda):
    """Another stream than the tensors' own; two captured graphs replayed at once, with new logits in place."""
    from nebulasd_b200.logprobs import token_logprobs
    sets = [_logits(20 + i, 16, 20000, torch.float16, cuda) for i in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_logprobs(*sets[0], 4)
    torch.cuda.current_stream().wait_stream(side)
    want = token_logprobs(*sets[0], 4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for logits, tokens in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(token_logprobs(logits, tokens, 4))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(3):
        for i, (logits, tokens) in enumerate(sets):
            x, t = _logits(40 + 2 * turn + i, 16, 20000, torch.float16, cuda)
            logits.copy_(x)
            tokens.copy_(t)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (logits, tokens), out in zip(sets, outs):
            assert all(torch.equal(a, b) for a, b in zip(out, token_logprobs(logits, tokens, 4)))


def test_two_calls_at_once(cuda):
    """Calls on two streams share nothing but the error word."""
    from nebulasd_b200.logprobs import token_logprobs, workspace_errors
    sets = [_logits(60 + i, rows, vocab, dtype, cuda)
            for i, (rows, vocab, dtype) in enumerate([(5, 151936, torch.float16), (300, 9001, torch.float32)])]
    want = [token_logprobs(x, t, 20) for x, t in sets]
    torch.cuda.synchronize()
    workspace_errors()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(token_logprobs(*sets[i], 20))
    torch.cuda.synchronize()
    for one, all_of in zip(want, got):
        assert all(torch.equal(a, b) for g in all_of for a, b in zip(g, one))
    assert workspace_errors() == 0


@pytest.mark.parametrize("dtype,rows", [(torch.bfloat16, 460), (torch.float16, 80)])
def test_whole_vocabulary_batches(dtype, rows, cuda):
    """More rows than the GPU holds at once, and a verify batch, against 64-bit torch on the GPU."""
    from nebulasd_b200.logprobs import token_logprobs
    vocab = 151936
    g = torch.Generator(device=cuda).manual_seed(rows)
    logits = (torch.randn((rows, vocab), generator=g, device=cuda) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=cuda).to(torch.int32)
    tokens[::2] = logits.argmax(1)[::2].to(torch.int32)
    tokens[5] = -1
    got = token_logprobs(logits, tokens, 32)
    for r in range(0, rows, 20):
        x, t = logits[r:r + 20].double(), tokens[r:r + 20].long()
        logp = torch.log_softmax(x, 1)
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :32]
        assert torch.equal(got.top_ids[r:r + 20].long(), ids)
        _close(got.top_logprobs[r:r + 20], logp.gather(1, ids).cpu(), vocab)
        _close(got.entropy[r:r + 20], -(logp.exp() * logp).sum(1).cpu(), vocab)
        own = t.clamp(min=0)[:, None]
        given = torch.where(t >= 0, logp.gather(1, own)[:, 0], math.nan)
        _close(got.logprobs[r:r + 20], given.cpu(), vocab)
        ranks = torch.where(t >= 0, 1 + (x > x.gather(1, own)).sum(1), 0)
        assert torch.equal(got.ranks[r:r + 20].long(), ranks)


def test_empty_batch(cuda):
    from nebulasd_b200.logprobs import token_logprobs
    got = token_logprobs(torch.empty((0, 100), dtype=torch.float16, device=cuda),
                         torch.empty(0, dtype=torch.int32, device=cuda), 3)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0,), (0, 3), (0, 3)]


def test_refusals_on_the_device(cuda):
    from nebulasd_b200.logprobs import token_logprobs
    x = torch.zeros((4, 100), dtype=torch.float16, device=cuda)
    t = torch.zeros(4, dtype=torch.int32, device=cuda)
    for args in ((x.t(), None, 0), (x, t.long(), 0), (x, t[:3], 0), (x, t[::2], 0), (x, t.cpu(), 0), (x, None, 33),
                 (x[:, :5], None, 6), (x, None, -1), (x.double(), None, 0), (x[:, :0], None, 0)):
        with pytest.raises(ValueError):
            token_logprobs(*args)
    for shape in ((1 << 31, 1), (1, (1 << 30) + 1)):  # (one element in memory)
        with pytest.raises(ValueError):
            token_logprobs(x[:1, :1].as_strided(shape, (0, 1) if shape[1] == 1 else (1 << 30, 0)))
