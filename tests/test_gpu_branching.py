"""GPU: a branching decode with all of its operators, as a program would run it.

Each round: decode attention over the pool, logits from its output, alternatives and log probabilities,
two branches forked per sequence without a host sync, each with its own next token stored, the less
likely rows freed, the pool compacted.  After each step the attention over the paged rows has to equal
the oracle's over every row's own, unshared history (fp16 outputs, the bar of the attention tests).
"""
import types

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_branches_over_a_shared_cache(cuda):
    from nebulasd_b200.block_pool import BlockPool
    from nebulasd_b200.kernels import store_kvcache
    from nebulasd_b200.kernels.paged_attn import paged_attention_raw
    from nebulasd_b200.logprobs import token_logprobs
    heads, kv_heads, dim, layers, vocab = 16, 8, 128, 2, 5003
    rows, width, num_blocks, seqs, keep = 12, 8, 64, 3, 1
    g = torch.Generator().manual_seed(1)
    emb_k, emb_v = (torch.randn((vocab, kv_heads, dim), generator=g).half() for _ in range(2))
    head = (torch.randn((heads * dim, vocab), generator=g) * 0.2).half().to(cuda)
    query = torch.randn((heads, dim), generator=g).half().to(cuda)
    k = torch.zeros((num_blocks, layers, kv_heads, 16, dim), dtype=torch.float16, device=cuda)
    v = torch.zeros_like(k)
    ints = lambda x: torch.tensor(list(x), dtype=torch.int32, device=cuda)  # noqa: E731
    pool = BlockPool(k, v, torch.full((rows, width), -1, dtype=torch.int32, device=cuda),
                     torch.zeros(rows, dtype=torch.int32, device=cuda),
                     torch.zeros(num_blocks, dtype=torch.int32, device=cuda))
    model = types.SimpleNamespace(num_q_heads=heads, num_kv_heads=kv_heads, head_dim=dim)
    engine = types.SimpleNamespace(block_size=16, max_blocks_per_seq=width)
    history = {r: [] for r in range(rows)}
    score = {}

    def store(at, tokens, lens):
        st = types.SimpleNamespace(num_prefill_seqs=0, num_prefill_tokens=0, num_decoding_seqs=len(at),
                                   prefill_seq_start_locs=None, prefill_seq_lens=None, seq_ids=ints(at),
                                   decoding_seq_lens=ints(lens))
        for layer in range(layers):
            store_kvcache(emb_k[tokens].to(cuda).contiguous(), emb_v[tokens].to(cuda).contiguous(), pool.k_cache,
                          pool.v_cache, pool.block_table, model, engine, st, layer)

    def attend(at):
        out = torch.empty((len(at), heads, dim), dtype=torch.float16, device=cuda)
        paged_attention_raw(query.expand(len(at), -1, -1).contiguous(), pool.k_cache, pool.v_cache, pool.block_table,
                            ints(len(history[r]) for r in at), ints(at), layers - 1, dim ** -0.5, out)
        for i, r in enumerate(at):
            kk = emb_k[history[r]].float().repeat_interleave(heads // kv_heads, 1)
            vv = emb_v[history[r]].float().repeat_interleave(heads // kv_heads, 1)
            p = torch.softmax(torch.einsum("hd,thd->ht", query.cpu().float(), kk) * dim ** -0.5, 1)
            want = torch.einsum("ht,thd->hd", p, vv)
            got = out[i].cpu().float()
            assert bool(((got - want).abs() <= 2e-3 + 1e-2 * want.abs()).all())
        return out

    # prompts of 15, 16 and 40 tokens
    prompts = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (15, 16, 40)]
    live = list(range(seqs))
    pool.fork(ints([0] * seqs), ints(live), ints([0] * seqs), ints(len(p) for p in prompts))
    for r, p in zip(live, prompts):
        for i, t in enumerate(p):
            history[r].append(t)
            store([r], [t], [i + 1])
        score[r] = 0.0
    origin = {r: r for r in live}
    for _ in range(6):
        out = attend(live)
        logits = out.reshape(len(live), -1) @ head
        got = token_logprobs(logits, None, 2)
        # Two children of every row, each with room for its next token; the parents go.
        parents = [r for r in live for _ in range(2)]
        empty = [r for r in range(rows) if r not in live][:len(parents)]
        lens = [len(history[r]) for r in parents]
        pool.fork(ints(parents), ints(empty), ints(lens), ints(n + 1 for n in lens))
        pool.free(ints(live))
        tokens, gains = got.top_ids.reshape(-1).tolist(), got.top_logprobs.reshape(-1).tolist()
        assert pool.errors() == 0
        for i, (p, c) in enumerate(zip(parents, empty)):
            history[c] = history[p] + [tokens[i]]
            score[c], origin[c] = score[p] + gains[i], origin[p]
        store(empty, tokens, [len(history[c]) for c in empty])
        attend(empty)
        # Each prompt keeps its best branches.
        kept = []
        for s in range(seqs):
            kept += sorted((c for c in empty if origin[c] == s), key=lambda c: -score[c])[:keep]
        pool.free(ints(c for c in empty if c not in kept))
        live = kept
        pool.compact()
        assert pool.errors() == 0
        attend(live)
        refs = pool.ref_counts.cpu().numpy()
        table, held = pool.block_table.cpu().numpy(), pool.seq_blocks.cpu().numpy()
        want = np.bincount(np.concatenate([table[r, :held[r]] for r in range(rows)]), minlength=num_blocks)
        assert np.array_equal(refs, want) and int((refs > 0).sum()) == refs.nonzero()[0].max() + 1
