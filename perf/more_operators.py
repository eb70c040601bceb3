"""Cases that measure a step of speculative decoding on a key / value cache held in 8 bits.

Five operators, in the order a step uses them:

* ``tables``  pages taken from and given back to the pool's free stack, page table, row ranges,
              positions and slots of a step, from the requests' lengths;
* ``store``   RMSNorm and rotation of the query and key heads, keys and values quantised to e4m3 with
              one power of two per page of 16 tokens and kv head, appended to the page pool;
* ``attend``  softmax attention over that pool: single tokens, the rows of drafted tokens, chunks;
* ``probs``   softmax of logits with a temperature for each row;
* ``verify``  drafted tokens accepted or rejected against the target's probabilities from given
              uniform numbers, and the token that follows the accepted ones.

``run`` computes a case with elementary torch operations, or, where ``own`` is true, with the
framework's entry points (``msgl.ops``). ``exact`` restates the definitions in 64 bits.

The pool's format: kv8 [pages, Hkv, 4096] e4m3 codes; the first 2048 of a page and head are the keys as
[2 halves of the dimensions][16 tokens][64], the others the values as [32 groups of 4 dimensions]
[4 groups c of tokens][4 dimensions][4 tokens 2c, 2c + 1, 8 + 2c, 9 + 2c]. scales [pages, Hkv, 2]: the
exponents of keys and values, 127 added. A value is code * 2^(scale - 127).
"""
import math
import os
import random
import sys

import torch

own = False

PAGE, HD = 16, 128
EPS = 1e-6
MAX_POSITION = 32768
FLOOR = 31  # smallest stored exponent: 2^-96
HEADS = [(16, 8), (32, 8), (32, 4), (8, 1), (64, 8)]  # query / kv heads (the last but one: a TP8 rank)
F8 = torch.float8_e4m3fn


def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _ops():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "mini-sglang-cpp_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from msgl import ops
    return ops


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a batch of requests that verify five drafted tokens each, and its way back after rejections
        dict(name="tables_verify_b64", op="tables", reqs=64, new_lo=6, new_hi=6, ctx=8000, back="accepted"),
        # prompts of 24 requests admitted at once, some of a cached prefix; all of them finish
        dict(name="tables_prompts", op="tables", reqs=24, new_lo=512, new_hi=4999, ctx=700, back="all"),
        # drafted rows of 48 requests behind the split-K qkv projection
        dict(name="store_verify_partials", op="store", reqs=48, chunk=5, ctx=4096, hq=32, hkv=8, parts=6),
        # chunks of two long prompts
        dict(name="store_prompts", op="store", reqs=2, chunk=4999, ctx=12000, hq=32, hkv=8, parts=0),
        # one request of a small model, one token
        dict(name="attend_one_4k", op="attend", reqs=1, chunk=1, ctx_lo=4099, ctx_hi=4099, hq=16, hkv=8),
        # a decode batch of ragged contexts
        dict(name="attend_decode_b128", op="attend", reqs=128, chunk=1, ctx_lo=1000, ctx_hi=4096, hq=32, hkv=8),
        # five drafted tokens and the last one of 24 requests at long contexts
        dict(name="attend_verify_b24", op="attend", reqs=24, chunk=6, ctx_lo=5000, ctx_hi=20000, hq=32, hkv=4),
        # chunks of two prompts whose earlier part is cached already
        dict(name="attend_chunks", op="attend", reqs=2, chunk=2048, ctx_lo=6000, ctx_hi=8192, hq=32, hkv=8),
        # the next token of one request
        dict(name="probs_one_row", op="probs", rows=1, vocab=151936),
        # target rows of 64 requests with four drafted tokens each
        dict(name="probs_verify_b64", op="probs", rows=320, vocab=151936),
        # one request
        dict(name="verify_one", op="verify", reqs=1, drafts=4, vocab=151936, point=False),
        # the same 64 requests
        dict(name="verify_b64", op="verify", reqs=64, drafts=4, vocab=151936, point=False),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "store", "attend", "attend", "probs", "verify"])
    if op == "tables":
        reqs = _log(rng, 1, 1024)
        hi = _log(rng, 1, min(8192, 65536 // reqs))
        return dict(op=op, reqs=reqs, new_lo=rng.choice([0, 1, (hi + 1) // 2, hi]) if hi > 1 else 1, new_hi=hi,
                    ctx=_log(rng, 1, 8192), back=rng.choice(["accepted", "all"]))
    if op == "store":
        hq, hkv = rng.choice(HEADS[:4])
        parts = rng.choice([0, 0, 1, 3, 6, 9])
        reqs = _log(rng, 1, 128)
        chunk = _log(rng, 1, max(1, (256 if parts else 8192) // reqs))
        return dict(op=op, reqs=reqs, chunk=chunk, ctx=chunk + _log(rng, 1, 8192), hq=hq, hkv=hkv, parts=parts)
    if op == "attend":
        hq, hkv = rng.choice(HEADS)
        kind = rng.random()
        if kind < 0.7:
            reqs = _log(rng, 1, 128)
            hi = _log(rng, 64, min(65536, (1 << 18) // reqs))
            chunk = 1 if kind < 0.4 else _log(rng, 2, 16)
        else:
            reqs = _log(rng, 1, 8)
            chunk, hi = _log(rng, 17, 2048 // reqs), _log(rng, 600, 8192)
            hq = 32 if hq == 64 else hq
        return dict(op=op, reqs=reqs, chunk=chunk, ctx_lo=max(chunk, hi // _log(rng, 1, 8)), ctx_hi=max(chunk, hi),
                    hq=hq, hkv=hkv)
    vocab = rng.choice([rng.randint(1000, 4000), 32000, 50257, 128256, 151936])
    if op == "probs":
        return dict(op=op, rows=_log(rng, 1, min(1024, 320 * 151936 // vocab)), vocab=vocab)
    return dict(op=op, reqs=_log(rng, 1, 64), drafts=rng.randint(0, 4), vocab=vocab, point=rng.random() < 0.3)


def _spread(n, lo, hi):
    """n whole numbers spread over [lo, hi], the first one hi."""
    return [hi - int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _rows(case):
    """New rows of each request: chunks are ragged, single tokens and drafted ones (up to 16) are not."""
    c = case["chunk"]
    return [c] * case["reqs"] if c <= 16 else _spread(case["reqs"], (c + 1) // 2, c)


def _contexts(case):
    q = _rows(case)
    lo, hi = (max(q), case["ctx"]) if case["op"] == "store" else (case["ctx_lo"], case["ctx_hi"])
    return [max(a, b) for a, b in zip(q, _spread(case["reqs"], lo, max(lo, hi)))]


# ------------------------------------------------------------------ inputs
def _normal(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen, device=gen.device) * std).to(dtype)


def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _table(dev):
    inv = 1e6 ** (-torch.arange(HD // 2, dtype=torch.float64, device=dev) / (HD // 2))
    ang = torch.arange(MAX_POSITION, dtype=torch.float64, device=dev)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _indptr(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _pages(lens, rng, extra):
    """A page table of `lens` tokens on pages in random order, and the pool's page count."""
    need = [-(-n // PAGE) for n in lens]
    ids = list(range(sum(need) + extra))
    rng.shuffle(ids)
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n] + [0] * (max(need) - n))
        at += n
    return rows, len(ids)


def _exponent(amax):
    """Smallest e with amax <= 448 * 2^e (448: the largest e4m3 value), as it is stored."""
    f, x = torch.frexp(amax)
    return torch.where(amax > 0, x - 9 + (f > 0.875).to(x.dtype) + 127, 0).clamp(min=FLOOR)


def _token_of_place(dev):
    """Token at place 4 c + e of a group of 4 dimensions."""
    i = torch.arange(PAGE, device=dev)
    return i % 4 // 2 * 8 + i // 4 * 2 + i % 2


def _place_of_token(dev):
    t = torch.arange(PAGE, device=dev)
    return t % 8 // 2 * 4 + t // 8 * 2 + t % 2


def _pack(k, v):
    """Codes [n, Hkv, 4096] of page keys and values [n, Hkv, 16 tokens, 128] (e4m3)."""
    n, h = k.shape[:2]
    k = k.view(torch.uint8).view(n, h, PAGE, 2, HD // 2).transpose(2, 3).reshape(n, h, -1)
    v = v.view(torch.uint8)[:, :, _token_of_place(v.device)]
    v = v.view(n, h, 4, 4, HD // 4, 4).permute(0, 1, 4, 2, 5, 3).reshape(n, h, -1)
    return torch.cat([k, v], 2)


def _unpack(codes):
    """Keys and values [n, Hkv, 16 tokens, 128] (e4m3) of codes [n, Hkv, 4096]."""
    n, h = codes.shape[:2]
    k = codes[:, :, :2048].reshape(n, h, 2, PAGE, HD // 2).transpose(2, 3).reshape(n, h, PAGE, HD)
    v = codes[:, :, 2048:].reshape(n, h, HD // 4, 4, 4, 4).permute(0, 1, 3, 5, 2, 4).reshape(n, h, PAGE, HD)
    v = v[:, :, _place_of_token(v.device)]
    return k.contiguous().view(F8), v.contiguous().view(F8)


def _power(stored):
    return torch.ldexp(torch.ones(stored.shape, device=stored.device), stored.int() - 127)


def _quantise(x):
    """Codes (e4m3) of pages x [n, Hkv, 16, 128] (fp32) and their stored exponents [n, Hkv]."""
    e = _exponent(torch.nan_to_num(x, nan=0.0).abs().amax((2, 3)))
    return (x / _power(e)[:, :, None, None]).to(F8), e.to(torch.uint8)


def _filled_pool(gen, pages, hkv):
    """A pool as a trained model fills it: keys with a few dimensions of large mean, pages of unlike size."""
    kv8 = torch.empty(pages, hkv, 4096, dtype=torch.uint8, device=gen.device)
    scales = torch.empty(pages, hkv, 2, dtype=torch.uint8, device=gen.device)
    mean = torch.zeros(HD, device=gen.device)
    mean[5], mean[69], mean[120] = 4.0, -5.0, 2.5
    for a in range(0, pages, 4096):
        n = min(4096, pages - a)
        x = torch.randn(2, n, hkv, PAGE, HD, generator=gen, device=gen.device)
        size = 2.0 ** torch.randint(-1, 2, (n, hkv, 1, 1), generator=gen, device=gen.device)
        (k, ke), (v, ve) = _quantise(x[0] + mean), _quantise(x[1] * size)
        kv8[a:a + n], scales[a:a + n] = _pack(k, v), torch.stack([ke, ve], 2)
    return kv8, scales


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    st = {"case": case}
    if case["op"] == "tables":
        B, hi = case["reqs"], case["new_hi"]
        new = _spread(B, case["new_lo"], hi)
        kept = [rng.randint(0 if case["back"] == "all" else 1, case["ctx"]) for _ in range(B)]
        # pages that a request holds: those of its kept tokens, at times one more from the draft before
        held = [-(-a // PAGE) + (rng.random() < 0.2) for a in kept]
        back = [a + rng.randint(min(1, n), n) if case["back"] == "accepted" else 0 for a, n in zip(kept, new)]
        width = -(-(case["ctx"] + hi) // PAGE) + 1
        ids = list(range(B * width))
        rng.shuffle(ids)
        rows = []
        for h in held:
            rows.append([ids.pop() for _ in range(h)] + [0] * (width - h))
        top = len(ids)
        free = ids + [-1] * (B * width - top)
        st.update(kept=_ints(kept, dev), new=_ints(new, dev), back=_ints(back, dev), none=_ints([0] * B, dev),
                  page_table=_ints(rows, dev).view(B, width), held=_ints(held, dev), free=_ints(free, dev),
                  top=_ints([top], dev), tokens=max(1, sum(new)) + 3)
    elif case["op"] == "store":
        lens, q_lens, hq, hkv = _contexts(case), _rows(case), case["hq"], case["hkv"]
        rows, pages = _pages(lens, rng, 3)
        T, nh = sum(q_lens), hq + 2 * hkv
        kv8, scales = _filled_pool(gen, pages, hkv)
        at = [n - q + i for n, q in zip(lens, q_lens) for i in range(q)]
        touched = [(r, p) for r, (n, q) in enumerate(zip(lens, q_lens)) for p in range((n - q) // PAGE, (n - 1) // PAGE + 1)]
        st.update(page_table=_ints(rows, dev), seq_lens=_ints(lens, dev), max_q=max(q_lens), kv8=kv8, scales=scales,
                  indptr=None if case["chunk"] == 1 else _ints(_indptr(q_lens), dev), positions=_ints(at, dev),
                  starts=_ints(_indptr(q_lens)[:-1], dev), rows=_ints(q_lens, dev), touched=torch.tensor(touched, device=dev),
                  table=_table(dev), qn=_normal(gen, HD, std=0.2).add_(1.0), kn=_normal(gen, HD, std=0.2).add_(1.0))
        if case["parts"]:
            st["parts"] = _normal(gen, case["parts"], T, nh * HD, std=case["parts"] ** -0.5, dtype=torch.float32)
        else:
            st["qkv"] = _normal(gen, T, nh * HD)
    elif case["op"] == "attend":
        lens, q_lens, hq, hkv = _contexts(case), _rows(case), case["hq"], case["hkv"]
        rows, pages = _pages(lens, rng, 3)
        kv8, scales = _filled_pool(gen, pages, hkv)
        st.update(page_table=_ints(rows, dev), seq_lens=_ints(lens, dev), max_seq=max(lens), max_q=max(q_lens), kv8=kv8,
                  scales=scales, indptr=None if case["chunk"] == 1 else _ints(_indptr(q_lens), dev),
                  of_token=torch.tensor([r for r, q in enumerate(q_lens) for _ in range(q)], device=dev),
                  row=torch.tensor([i for q in q_lens for i in range(q)], device=dev),
                  at=torch.tensor([n - q + i for n, q in zip(lens, q_lens) for i in range(q)], device=dev),
                  q=_normal(gen, sum(q_lens), hq, HD))
    else:
        V = case["vocab"]
        B, k = (case["rows"], 0) if case["op"] == "probs" else (case["reqs"], case["drafts"])
        T = B * (k + 1)
        logits = _normal(gen, T, V, std=2.5, dtype=torch.float32)
        # a few likely tokens a row
        likely = torch.randint(0, V, (T, 12), generator=gen, device=dev)
        logits.scatter_add_(1, likely, _normal(gen, T, 12, std=3.0, dtype=torch.float32) + 9.0)
        if case["op"] == "probs":
            temperature = torch.rand(T, generator=gen, device=dev) + 0.5
            if T > 2:
                temperature[1] = 0.0  # a greedy request
            st.update(logits=logits, temperature=temperature)
        else:
            p = torch.softmax(logits, 1)
            pick = torch.tensor([r * (k + 1) + i for r in range(B) for i in range(k)], dtype=torch.int64, device=dev)
            near = logits[pick] + _normal(gen, B * k, V, std=0.7, dtype=torch.float32)
            q = torch.softmax(near, 1)
            tokens = (q.argmax(1) if case["point"] else torch.multinomial(q, 1, generator=gen)[:, 0]) if B * k else pick
            st.update(p=p, q=None if case["point"] else q, tokens=tokens.int(),
                      indptr=_ints([r * k for r in range(B + 1)], dev), u=torch.rand(B * k, generator=gen, device=dev),
                      last=torch.rand(B, generator=gen, device=dev))
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    return {"tables": _run_tables, "store": _run_store, "attend": _run_attend, "probs": _run_probs,
            "verify": _run_verify}[st["case"]["op"]](st)


def _run_tables(st):
    pools = {"page_table": st["page_table"], "held": st["held"], "free": st["free"], "top": st["top"]}
    if own:
        ops = _ops()
        if "out" not in st:  # the buffers that a serving loop keeps
            B = st["kept"].numel()
            st["out"] = ops.step_tables_buffers(B, st["tokens"]), ops.step_tables_buffers(B, 0)
        step, back = st["out"]
        state = st["page_table"], st["held"], st["free"], st["top"]
        ops.step_tables(st["kept"], st["new"], *state, out=step)
        ops.step_tables(st["back"], st["none"], *state, out=back)
    else:
        step = _plain_tables(st, st["kept"], st["new"], st["tokens"])
        back = _plain_tables(st, st["back"], st["none"], 0)
    return {"step": list(step), "back": [back[0], back[1], back[4]], **pools}


def _plain_tables(st, kept, new, tokens):
    """seq_lens, q_indptr, positions, slots, index of each request's last row; pages and free stack in place."""
    table, held, free, top = st["page_table"], st["held"], st["free"], st["top"]
    B, width = table.shape
    dev = table.device
    total = kept + new
    need = (total + PAGE - 1) // PAGE
    give, take = (held - need).clamp(min=0), (need - held).clamp(min=0)
    c = torch.arange(width, device=dev)
    at = top + (give.cumsum(0) - give)[:, None] + held[:, None] - 1 - c
    at = torch.where((c >= need[:, None]) & (c < held[:, None]), at, free.numel())
    free.copy_(torch.cat([free, free[:1]]).scatter(0, at.view(-1).long(), table.view(-1))[:-1])
    top = top + give.sum()
    at = top - 1 - (take.cumsum(0) - take)[:, None] - (c - held[:, None])
    new_page = (c >= held[:, None]) & (c < need[:, None])
    table.copy_(torch.where(new_page, free[at.clamp(0, free.numel() - 1).long()], table))
    st["top"].copy_(top - take.sum())
    held.copy_(need)
    indptr = torch.cat([new.new_zeros(1), new.cumsum(0, dtype=torch.int32)])
    t = torch.arange(tokens, device=dev)
    r = (t[:, None] >= indptr[None, 1:]).sum(1)
    live = r < B
    r = r.clamp(max=B - 1)
    pos = torch.where(live, kept[r] + t - indptr[r], 0)
    slot = torch.where(live, table[r, pos // PAGE] * PAGE + pos % PAGE, -1)
    return total, indptr, pos.int(), slot.int(), torch.where(new > 0, indptr[1:] - 1, -1)


def _run_store(st):
    case = st["case"]
    hq, hkv = case["hq"], case["hkv"]
    cache = {"kv8": st["kv8"].view(F8), "scales": st["scales"].view(torch.float8_e8m0fnu)}
    if own:
        ops = _ops()
        src, call = ((st["parts"], ops.qknorm_rope_store_kv8_partials) if case["parts"]
                     else (st["qkv"], ops.qknorm_rope_store_kv8))
        if "out" not in st:  # kept by a serving loop
            st["out"] = torch.empty(st["positions"].numel(), hq, HD, dtype=torch.bfloat16, device=src.device)
        q = call(src, st["kv8"], st["scales"], st["positions"], st["page_table"], st["seq_lens"], st["table"], st["qn"],
                 st["kn"], hq, hkv, EPS, q_indptr=st["indptr"], max_q_len=st["max_q"], out=st["out"])
        return {"q": q, **cache}
    x = st["parts"].sum(0) if case["parts"] else st["qkv"].float()
    x = x.view(x.shape[0], hq + 2 * hkv, HD)
    qk, v = x[:, :hq + hkv], x[:, hq + hkv:]
    w = torch.cat([st["qn"].float().expand(hq, HD), st["kn"].float().expand(hkv, HD)])
    qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * w
    turn = st["table"][st["positions"].long()][:, None]
    c, s = turn[..., :HD // 2], turn[..., HD // 2:]
    lo, hi = qk[..., :HD // 2], qk[..., HD // 2:]
    qk = torch.cat([lo * c - hi * s, lo * s + hi * c], -1)
    # the touched pages: earlier tokens as they are held, new ones, zeros behind the context's end
    r, page = st["touched"].T
    phys = st["page_table"].long()[r, page]
    i = page[:, None] * PAGE + torch.arange(PAGE, device=r.device) - (st["seq_lens"] - st["rows"])[r][:, None]
    n = st["rows"][r][:, None]
    row = (st["starts"][r][:, None] + i.clamp(min=0)).clamp(max=x.shape[0] - 1)
    scale = _power(st["scales"][phys])
    pages = []
    for old, fresh, e in zip(_unpack(st["kv8"][phys]), (qk[:, hq:], v), scale.unbind(2)):
        old = old.float() * e[:, :, None, None]
        fresh = fresh[row].transpose(1, 2)
        pages.append(_quantise(torch.where((i < 0)[:, None, :, None], old, torch.where((i < n)[:, None, :, None], fresh, 0.0))))
    (kc, ke), (vc, ve) = pages
    st["kv8"][phys] = _pack(kc, vc)
    st["scales"][phys] = torch.stack([ke, ve], 2)
    return {"q": qk[:, :hq].to(torch.bfloat16), **cache}


def _run_attend(st):
    case = st["case"]
    hq, hkv = case["hq"], case["hkv"]
    if own:
        ops = _ops()
        if "ws" not in st:  # the workspace and the output buffer that a serving loop keeps
            T = st["q"].shape[0]
            st["ws"] = ops.attention_kv8_workspace(case["reqs"], st["max_q"], hq, hkv)
            st["out"] = torch.empty(T, hq, HD, dtype=torch.bfloat16, device=st["q"].device)
        return ops.paged_attention_kv8(st["q"], st["kv8"], st["scales"], st["page_table"], st["seq_lens"], st["max_seq"],
                                       hq, hkv, q_indptr=st["indptr"], max_q_len=st["max_q"], workspace=st["ws"],
                                       out=st["out"])
    q, of, row, at = st["q"], st["of_token"], st["row"], st["at"]
    T, G, B, n = q.shape[0], hq // hkv, case["reqs"], st["max_q"]
    phys = st["page_table"].long()
    P = phys.shape[1]
    e = _power(st["scales"][phys.view(-1)])
    k, v = ((c.float() * e[:, :, j, None, None]).view(B, P, hkv, PAGE, HD).transpose(1, 2).reshape(B, hkv, P * PAGE, HD)
            for j, c in enumerate(_unpack(st["kv8"][phys.view(-1)])))
    qp = torch.zeros(B, n, hkv, G, HD, device=q.device)
    qp[of, row] = q.view(T, hkv, G, HD).float()
    end = torch.full((B, n), -1, device=q.device)
    end[of, row] = at
    s = qp.permute(0, 2, 1, 3, 4).reshape(B, hkv, n * G, HD) @ k.transpose(2, 3) * HD ** -0.5
    seen = torch.arange(P * PAGE, device=q.device) <= end.repeat_interleave(G, 1)[:, None, :, None]
    s = torch.where(seen, s, -math.inf)
    s = (s - s.amax(-1, keepdim=True)).exp()
    s = (s / s.sum(-1, keepdim=True)) @ v
    s = s.view(B, hkv, n, G, HD).transpose(1, 2)[of, row]
    return s.reshape(T, hq, HD).to(torch.bfloat16)


def _run_probs(st):
    if own:
        ops = _ops()
        if "out" not in st:
            st["out"] = torch.empty_like(st["logits"])
        return ops.token_probs(st["logits"], st["temperature"], out=st["out"])
    x, t = st["logits"], st["temperature"][:, None]
    top = x.amax(1, keepdim=True)
    e = ((x - top) / torch.where(t > 0, t, 1.0)).exp()
    e = e / e.sum(1, keepdim=True)
    first = torch.arange(x.shape[1], device=x.device) == x.argmax(1, keepdim=True)
    return torch.where(t > 0, e, first.float())


def _run_verify(st):
    case = st["case"]
    if own:
        ops = _ops()
        if "out" not in st:
            B, dev = case["reqs"], st["p"].device
            st["out"] = (torch.empty(B, dtype=torch.int32, device=dev),
                         torch.empty(B, case["drafts"] + 1, dtype=torch.int32, device=dev))
        return ops.verify_drafts(st["p"], st["q"], st["tokens"], st["indptr"], st["u"], st["last"], case["drafts"],
                                 out=st["out"])
    B, k, V = case["reqs"], case["drafts"], case["vocab"]
    dev = st["p"].device
    p, x = st["p"].view(B, k + 1, V), st["tokens"].long().view(B, k)
    r = torch.arange(B, device=dev)
    px = p[:, :k].gather(2, x[..., None])[..., 0]
    if st["q"] is None:
        qx = torch.ones_like(px)
    else:
        q = st["q"].view(B, k, V)
        qx = q.gather(2, x[..., None])[..., 0]
    ok = st["u"].double().view(B, k) * qx.double() < px.double()
    n = ok.long().cumprod(1).sum(1)  # accepted
    w = p[r, n].double()
    if k:
        at = n.clamp(max=k - 1)
        if st["q"] is None:
            other = (torch.arange(V, device=dev) == x[r, at][:, None]).double()
        else:
            other = q[r, at].double()
        rest = (w - other * (n < k)[:, None]).clamp(min=0)
        w = torch.where(rest.sum(1, keepdim=True) > 0, rest, w)
    c = w.cumsum(1)
    token = (c <= st["last"].double()[:, None] * c[:, -1:]).sum(1)
    i = torch.arange(k + 1, device=dev)
    tokens = torch.where(i < n[:, None], torch.cat([x, x.new_zeros(B, 1)], 1), -1)
    tokens = torch.where(i == n[:, None], token[:, None], tokens)
    return n.int(), tokens.int()


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "tables":
        tokens = sum(_spread(case["reqs"], case["new_lo"], case["new_hi"]))
        return {"bytes": tokens * 8 + case["reqs"] * 2 * 28 + 2 * 8 * (tokens / PAGE + case["reqs"]), "flops": tokens * 4}
    if case["op"] == "store":
        lens, q = _contexts(case), _rows(case)
        T, nh = sum(q), case["hq"] + 2 * case["hkv"]
        pages = sum((n - 1) // PAGE - (n - m) // PAGE + 1 for n, m in zip(lens, q))
        old = sum((n - m) % PAGE for n, m in zip(lens, q))  # earlier tokens of touched pages
        total = T * nh * HD * (4 * case["parts"] if case["parts"] else 2) + T * (HD * 4 + 4) + T * case["hq"] * HD * 2
        return {"bytes": total + case["hkv"] * (pages * 4096 + old * 256), "flops": 10.0 * T * nh * HD}
    if case["op"] == "attend":
        hq, hkv = case["hq"], case["hkv"]
        total, flops = 0.0, 0.0
        for n, m in zip(_contexts(case), _rows(case)):
            total += n * hkv * 256 + -(-n // PAGE) * (hkv * 2 + 4) + m * hq * HD * 4
            flops += 4.0 * HD * hq * (m * (n - m) + m * (m + 1) / 2)
        return {"bytes": total, "flops": flops}
    if case["op"] == "probs":
        return {"bytes": case["rows"] * (case["vocab"] * 8.0 + 4), "flops": case["rows"] * case["vocab"] * 4.0}
    rows = 1 if case["point"] else 2  # the target's and the draft's row of the final token
    return {"bytes": case["reqs"] * (rows * case["vocab"] * 4.0 + case["drafts"] * 20),
            "flops": case["reqs"] * case["vocab"] * 3.0}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"tables": _exact_tables, "store": _exact_store, "attend": _exact_attend, "probs": _exact_probs,
            "verify": _exact_verify}[case["op"]](st)


def _exact_tables(st):
    kept, new, back = (st[k].tolist() for k in ("kept", "new", "back"))
    indptr, pos = _indptr(new), [a + i for a, n in zip(kept, new) for i in range(n)]
    pos += [0] * (st["tokens"] - len(pos))
    last = [e - 1 if n else -1 for e, n in zip(indptr[1:], new)]
    whole = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    # which pages they are depends on the passes before
    return {"step": [whole([a + n for a, n in zip(kept, new)]), whole(indptr), whole(pos), None, whole(last)],
            "back": [whole(back), whole([0] * len(new) + [0]), whole([-1] * len(new))],
            "page_table": None, "held": whole([-(-a // PAGE) for a in back]), "free": None, "top": None}


def _e4m3(x):
    """x rounded to the nearest e4m3 value, ties to the even one (|x| <= 448), in 64 bits."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def _exact_store(st):
    case = st["case"]
    hq, hkv = case["hq"], case["hkv"]
    x = (st["parts"].double().sum(0) if case["parts"] else st["qkv"].double()).view(-1, hq + 2 * hkv, HD)
    w = torch.cat([st["qn"].double().expand(hq, HD), st["kn"].double().expand(hkv, HD)])
    y = x[:, :hq + hkv]
    y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / HD + EPS) * w
    row = st["table"].double()[st["positions"].long()]
    z = torch.empty_like(y)
    for d in range(HD // 2):
        c, s = row[:, d, None], row[:, d + HD // 2, None]
        z[..., d] = y[..., d] * c - y[..., d + HD // 2] * s
        z[..., d + HD // 2] = y[..., d] * s + y[..., d + HD // 2] * c
    kv8, scales = st["kv8"].view(F8).double(), torch.exp2(st["scales"].double() - 127)
    pages = st["page_table"].tolist()
    dim, tok = torch.arange(HD, device=x.device), torch.arange(PAGE, device=x.device)[:, None]
    place = (dim // 64 * 1024 + tok * 64 + dim % 64,
             2048 + dim // 4 * 64 + tok % 8 // 2 * 16 + dim % 4 * 4 + tok // 8 * 2 + tok % 2)
    touched = st["touched"].tolist()
    lens, rows, starts = st["seq_lens"].tolist(), st["rows"].tolist(), st["starts"].tolist()
    for j, new in ((0, z[:, hq:]), (1, x[:, hq + hkv:])):
        values = torch.zeros(len(touched), hkv, PAGE, HD, dtype=torch.float64, device=x.device)
        for a, (r, p) in enumerate(touched):
            begin = lens[r] - rows[r]
            old = min(PAGE, max(0, begin - p * PAGE))
            phys, end = pages[r][p], min(lens[r], (p + 1) * PAGE)
            if old:
                values[a, :, :old] = kv8[phys][:, place[j][:old]] * scales[phys, :, j, None, None]
            first = max(begin, p * PAGE)
            take = starts[r] + first - begin
            values[a, :, first - p * PAGE:end - p * PAGE] = new[take:take + end - first].transpose(0, 1)
        top = values.abs().amax((2, 3))
        e = torch.where(top > 0, torch.ceil(torch.log2(top.clamp(min=1e-300) / 448)), -96.0).clamp(min=-96)
        e = torch.where(top > 448 * torch.exp2(e), e + 1, torch.where((top <= 448 * torch.exp2(e - 1)) & (e > -96), e - 1, e))
        codes = _e4m3(values / torch.exp2(e)[:, :, None, None])
        at = torch.tensor([pages[r][p] for r, p in touched], device=x.device)
        kv8[at[:, None, None, None], torch.arange(hkv, device=x.device)[:, None, None], place[j]] = codes
        scales[at, :, j] = torch.exp2(e)
    return {"q": z[:, :hq], "kv8": kv8, "scales": scales}


def _exact_attend(st):
    case = st["case"]
    hq, hkv = case["hq"], case["hkv"]
    G = hq // hkv
    out = torch.zeros(st["q"].shape[0], hq, HD, dtype=torch.float64, device=st["q"].device)
    t = 0
    for r, (n, m) in enumerate(zip(_contexts(case), _rows(case))):
        phys = st["page_table"][r, :-(-n // PAGE)].long()
        codes = _unpack(st["kv8"][phys])
        e = torch.exp2(st["scales"][phys].double() - 127)
        hidden = torch.arange(n, device=phys.device) > torch.arange(n - m, n, device=phys.device)[:, None]
        for h in range(hkv):
            key, val = ((c[:, h].double() * e[:, h, j, None, None]).reshape(-1, HD)[:n] for j, c in enumerate(codes))
            for g in range(h * G, (h + 1) * G):
                s = (st["q"][t:t + m, g].double() @ key.T / math.sqrt(HD)).masked_fill(hidden, -math.inf)
                out[t:t + m, g] = torch.softmax(s, -1) @ val
        t += m
    return out


def _exact_probs(st):
    out = torch.empty_like(st["logits"], dtype=torch.float64)
    for i, t in enumerate(st["temperature"].double().tolist()):
        x = st["logits"][i].double()
        if t > 0:
            out[i] = torch.softmax(x / t, 0)
        else:
            out[i] = 0
            out[i, int((x == x.max()).nonzero()[0])] = 1
    return out


def _exact_verify(st):
    case = st["case"]
    B, k = case["reqs"], case["drafts"]
    counts, rows = [], []
    for r in range(B):
        got = []
        for i in range(k):
            x = int(st["tokens"][r * k + i])
            q = 1.0 if st["q"] is None else float(st["q"][r * k + i, x])
            if not float(st["u"][r * k + i]) * q < float(st["p"][r * (k + 1) + i, x]):
                break
            got.append(x)
        n = len(got)
        w = st["p"][r * (k + 1) + n].double()
        if n < k:
            rest = w.clone()
            if st["q"] is None:
                rest[int(st["tokens"][r * k + n])] -= 1
            else:
                rest -= st["q"][r * k + n].double()
            rest = torch.where(rest > 0, rest, 0.0)
            w = rest if bool((rest > 0).any()) else w
        sums = torch.cumsum(w, 0)
        got.append(int(torch.searchsorted(sums, float(st["last"][r]) * sums[-1], right=True)))
        counts.append(n)
        rows.append(got + [-1] * (k + 1 - len(got)))
    return [torch.tensor(counts, dtype=torch.int32), torch.tensor(rows, dtype=torch.int32)]
