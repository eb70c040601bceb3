"""A speculative decoding loop over the 8-bit pool on a B200: tables, append, attention, probabilities and verification
as a server calls them, with a random projection for the model; every step against 64-bit restatements and the page
pool's own bookkeeping on lists. Tolerances as in the operators' own tests."""
import random

import pytest
import torch

from kv8_plain import D, PAGE, ints, pool_values
from test_kv8_gpu import EPS, Attend, table, turned
from test_step_tables_gpu import Pool
from test_verify_gpu import check_probs, restate

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,drafts,hq,hkv", [(1, 3, 8, 2), (5, 4, 8, 1), (3, 0, 4, 4), (9, 7, 16, 8)])
def test_loop(cuda, B, drafts, hq, hkv):
    from msgl import ops
    rng, g = random.Random(B), torch.Generator("cuda").manual_seed(B)
    V, width, nh = 300, 24, hq + 2 * hkv
    pool = Pool(B, width, B * width, seed=B)
    kv8, scales = ops.kv8_pool(B * width, hkv)
    embed = torch.randn(V, nh * D, generator=g, device="cuda").bfloat16()      # a token's QKV row
    head = torch.randn(hq * D, V, generator=g, device="cuda") * 0.2
    qn, kn = ((1 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16() for _ in range(2))
    tab = table(width * PAGE)
    ws = ops.attention_kv8_workspace(B, 64, hq, hkv)
    history = [[rng.randrange(V) for _ in range(rng.randint(1, 60))] for _ in range(B)]  # all tokens, the last not yet run
    kept = [0] * B  # tokens whose keys and values are stored
    moved = 0
    for step in range(6):
        if step == 3:  # a request ends, another takes its place
            history[0], kept[0] = [rng.randrange(V) for _ in range(33)], 0
        # what the draft model proposes (none behind a prompt that is still to run)
        ks = [drafts if len(h) - k == 1 else 0 for h, k in zip(history, kept)]
        proposed = [[rng.randrange(V) for _ in range(k)] for k in ks]
        rows = [h[k:] + p for h, k, p in zip(history, kept, proposed)]
        new = [len(r) for r in rows]
        T = sum(new)
        got = pool.check(kept, new, T + 5)
        ids = torch.tensor([t for r in rows for t in r] + [0] * 5, device="cuda")
        qkv = embed[ids]
        q = torch.full((T + 5, hq, D), 7.0, device="cuda").bfloat16()
        kw = dict(q_indptr=got.q_indptr, max_q_len=max(new))
        ops.qknorm_rope_store_kv8(qkv, kv8, scales, got.positions, pool.table, got.seq_lens, tab, qn, kn, hq, hkv, EPS, out=q, **kw)
        assert bool((q[T:] == 7).all())
        # the whole context of every request: e4m3 of the formula
        for r in range(B):
            ctx = torch.tensor(history[r][:kept[r]] + rows[r], device="cuda")
            x = embed[ctx].double().view(-1, nh, D)
            w = torch.cat([qn.expand(hq, D), kn.expand(hkv, D)])
            ref, mag = turned(x[:, :hq + hkv], torch.arange(len(ctx), device="cuda"), tab, w)
            at = torch.tensor(pool.rows[r], device="cuda")
            for kind, want, off in ((0, ref[:, hq:], mag[:, hq:] * 2 ** -17), (1, x[:, hq + hkv:], 0.0)):
                held = pool_values(kv8[at], scales[at], kind).transpose(1, 2).reshape(-1, hkv, D)[:len(ctx)]
                s = torch.exp2(scales[at, :, kind].double() - 127).repeat_interleave(PAGE, 0)[:len(ctx), :, None]
                # half a step, and half of a subnormal one again for each time that the page was written before
                assert bool(((held - want).abs() <= torch.maximum(want.abs() * 2 ** -4, s * 2 ** -10) + s * 2 ** -10 * step + off * 1.07).all())
        out = ops.paged_attention_kv8(q, kv8, scales, pool.table, got.seq_lens, max(k + n for k, n in zip(kept, new)), hq, hkv, workspace=ws, **kw)
        a = Attend.__new__(Attend)
        a.lens, a.rows, a.hq, a.hkv, a.table, a.kv8, a.scales, a.q = [k + n for k, n in zip(kept, new)], new, hq, hkv, pool.table, kv8, scales, q
        a.check(out)
        # target rows: the last k + 1 of each request
        start = [sum(new[:r + 1]) - ks[r] - 1 for r in range(B)]
        pick = torch.tensor([s + i for s, k in zip(start, ks) for i in range(k + 1)], device="cuda")
        logits = out.view(-1, hq * D)[pick].float() @ head
        t = torch.tensor([0.0 if r % 4 == 3 else 0.9 for r, k in enumerate(ks) for _ in range(k + 1)], device="cuda")
        p = ops.token_probs(logits, t)
        warm = t > 0
        check_probs(p[warm], logits[warm], t[warm])
        assert torch.equal(p[~warm].argmax(1), logits[~warm].argmax(1)) and bool((p[~warm].sum(1) == 1).all())
        # drafts: likely tokens at times, so that some are accepted
        n = sum(ks)
        rowof = torch.tensor([sum(ks[:r]) + r + i for r in range(B) for i in range(ks[r])], dtype=torch.int64, device="cuda")
        dq = torch.softmax(torch.log(p[rowof] + 1e-4) + 0.3 * torch.randn(n, V, generator=g, device="cuda"), 1)
        toks = torch.tensor([x for pr in proposed for x in pr], dtype=torch.int32, device="cuda")
        indptr = ints([sum(ks[:r]) for r in range(B + 1)])
        u, last = torch.rand(n, generator=g, device="cuda") * 0.5, torch.rand(B, generator=g, device="cuda")
        acc, tokens = ops.verify_drafts(p, dq, toks, indptr, u, last, max(1, drafts))
        want_acc, want, sure = restate(p, dq, toks, indptr, u, last, max(1, drafts))
        assert acc.tolist() == want_acc and all(not ok or x == y for ok, x, y in zip(sure, tokens.tolist(), want))
        for r in range(B):
            done = tokens[r, :want_acc[r] + 1].tolist()
            kept[r] = len(history[r]) + want_acc[r]  # the last of `done` runs in the next step
            history[r] += done
            moved += want_acc[r]
            if kept[r] + drafts + 2 > width * PAGE:
                history[r], kept[r] = history[r][:5], 0
        assert ops.device_error() == (0, 0)
    assert moved > 0 or drafts == 0
    pool.check([0] * B, [0] * B, 0)
    assert sorted(pool.free) == list(range(B * width))
