"""Cases that measure the attention-side operators of long multi-axis contexts and of adapters.

Four operators of one decoder layer, in the order a step runs them:

* ``lora``    low-rank adapters of many requests beside a shared projection:
              d[t] = scale[a] * B[a] (A[a] x[t]) for the adapter a of t's request, added to the
              projection's bf16 output or written as one more fp32 split-K partial;
* ``store``   RMSNorm of every query and key head, rotation by positions of three axes (time,
              height, width), append of keys and values to the page pool;
* ``bounds``  smallest and largest key of every page that the step's tokens touched, per kv head
              and dimension;
* ``sparse``  pages selected per query and kv head by an upper bound of their attention logits,
              then softmax attention over the selected pages only; single tokens and chunks.

``run`` computes a case with elementary torch operations, or, where ``own`` is true, with the
framework's entry points (``msgl.ops``). ``exact`` restates the definitions in 64 bits.
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
HEADS = [(16, 8), (32, 8), (32, 4), (8, 1), (64, 8)]  # query / kv heads (the last but one: a TP8 rank)


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
        # one token of a small model, one adapter: the latency of two dependent small products
        dict(name="lora_one_token", op="lora", reqs=1, chunk=1, k=1024, n=4096, rank=16, adapters=4,
             partial=False),
        # a decode batch whose requests use 48 adapters on the 4096 -> 6144 qkv projection, which
        # itself runs as split-K partials: the adapters are one partial more
        dict(name="lora_decode_b128", op="lora", reqs=128, chunk=1, k=4096, n=6144, rank=16,
             adapters=48, partial=True),
        # prompts of six tenants in one chunk of about 4k tokens, high rank
        dict(name="lora_prompts_r64", op="lora", reqs=6, chunk=901, k=4096, n=6144, rank=64,
             adapters=5, partial=False),
        # one decoded token of a small model
        dict(name="store_one_token", op="store", tokens=1, hq=16, hkv=8, parts=0, s1=20, s2=20,
             interleaved=True),
        # a decode batch behind the split-K qkv projection
        dict(name="store_decode_b128_partials", op="store", tokens=128, hq=32, hkv=8, parts=6,
             s1=24, s2=24, interleaved=False),
        # a chunk of a video prompt
        dict(name="store_video_chunk", op="store", tokens=8191, hq=32, hkv=8, parts=0, s1=20, s2=20,
             interleaved=True),
        # decode: every request's last page changes
        dict(name="bounds_decode_b128", op="bounds", reqs=128, chunk=1, ctx_lo=1000, ctx_hi=4096,
             hkv=8),
        # chunks of four prompts: some 2k pages are completed
        dict(name="bounds_prompts", op="bounds", reqs=4, chunk=10001, ctx_lo=10001, ctx_hi=16384,
             hkv=8),
        # one request of a small model at a moderate context
        dict(name="sparse_one_4k", op="sparse", reqs=1, chunk=1, ctx_lo=4099, ctx_hi=4099, hq=16,
             hkv=8, top=32, sink=1, recent=2),
        # one request at a very long context
        dict(name="sparse_one_131k", op="sparse", reqs=1, chunk=1, ctx_lo=131067, ctx_hi=131067,
             hq=32, hkv=4, top=256, sink=1, recent=4),
        # a decode batch of long ragged contexts
        dict(name="sparse_decode_b64", op="sparse", reqs=64, chunk=1, ctx_lo=4096, ctx_hi=32768,
             hq=32, hkv=8, top=128, sink=1, recent=4),
        # chunks of three prompts whose earlier part is cached already
        dict(name="sparse_chunks", op="sparse", reqs=3, chunk=512, ctx_lo=6000, ctx_hi=16384,
             hq=32, hkv=8, top=64, sink=1, recent=4),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lora", "store", "bounds", "sparse"])
    if op == "lora":
        partial = rng.random() < 0.4
        reqs = _log(rng, 1, 128)
        chunk = _log(rng, 1, max(1, (256 if partial else 4096) // reqs))
        return dict(op=op, reqs=reqs, chunk=chunk, k=rng.choice([1000, 1024, 2048, 4096, 5120]),
                    n=rng.choice([1024, 2048, 2568, 4096, 5120, 6144]),
                    rank=rng.choice([8, 16, 24, 32, 64, 128] if reqs * chunk <= 1024 else [8, 16, 32, 64]),
                    adapters=_log(rng, 1, 48), partial=partial)
    if op == "store":
        hq, hkv = rng.choice(HEADS[:4])
        parts = rng.choice([0, 0, 1, 3, 6, 9])
        return dict(op=op, tokens=_log(rng, 1, 256 if parts else 8191), hq=hq, hkv=hkv, parts=parts,
                    s1=rng.randint(0, 21), s2=rng.randint(0, 21), interleaved=rng.random() < 0.5)
    if op == "bounds":
        reqs = _log(rng, 1, 128)
        chunk = 1 if rng.random() < 0.5 else _log(rng, 1, max(1, 32768 // reqs))
        lo = chunk + _log(rng, 1, 1024) - 1
        return dict(op=op, reqs=reqs, chunk=chunk, ctx_lo=lo, ctx_hi=lo + _log(rng, 1, 2048),
                    hkv=rng.choice([1, 4, 8]))
    hq, hkv = rng.choice(HEADS)
    if rng.random() < 0.6:
        reqs = _log(rng, 1, 64)
        hi = _log(rng, 64, min(65536, (1 << 20) // reqs))
        chunk, top = 1, _log(rng, 2, 256 if reqs <= 32 else 128)
    else:
        reqs = _log(rng, 1, 8)
        chunk, hi, top = _log(rng, 2, max(2, 1000 // reqs)), _log(rng, 1100, 12000), _log(rng, 2, 64)
        if hq == 64:
            hq = 32
    sink = rng.randint(0, min(2, top - 1))
    return dict(op="sparse", reqs=reqs, chunk=chunk, ctx_lo=max(chunk, hi // _log(rng, 1, 8)),
                ctx_hi=max(chunk, hi), hq=hq, hkv=hkv, top=top, sink=sink,
                recent=rng.randint(1, min(8, top - sink)))


def _spread(n, lo, hi):
    """n whole numbers spread over [lo, hi], the first one hi."""
    return [hi - int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _chunks(case):
    """New tokens of each request: 1 in decode, else a ragged half to the whole of `chunk`."""
    c = case["chunk"]
    return [1] * case["reqs"] if c == 1 else _spread(case["reqs"], (c + 1) // 2, c)


def _contexts(case):
    q = _chunks(case)
    return [max(a, b) for a, b in zip(q, _spread(case["reqs"], case["ctx_lo"], case["ctx_hi"]))]


def _axis_map(case):
    """Axis (0 time, 1 height, 2 width) whose position turns the rotary pair d, d = 0 .. 63."""
    half, s1, s2 = HD // 2, case["s1"], case["s2"]
    if case["interleaved"]:
        return [1 if d % 3 == 1 and d < 3 * s1 else 2 if d % 3 == 2 and d < 3 * s2 else 0
                for d in range(half)]
    s0 = half - s1 - s2
    return [0 if d < s0 else 1 if d < s0 + s1 else 2 for d in range(half)]


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


def _keys(gen, num_slots, hkv):
    """Keys as a trained cache holds them: unit noise, a few dimensions with a large mean."""
    k = torch.randn(num_slots, hkv, HD, generator=gen, device=gen.device, dtype=torch.float32
                    if num_slots * hkv < 1 << 20 else torch.bfloat16)
    mean = torch.zeros(hkv, HD, device=gen.device)
    mean[:, 5], mean[:, 69], mean[:, 120] = 4.0, -5.0, 2.5
    return k.add_(mean.to(k.dtype)).to(torch.bfloat16)


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    st = {"case": case}
    if case["op"] == "lora":
        lens = _chunks(case)
        T, K, N, R, n = sum(lens), case["k"], case["n"], case["rank"], case["adapters"]
        # about one request in eight runs the plain model
        ids = [-1 if rng.random() < 0.125 else rng.randrange(n) for _ in lens]
        ids[0] = rng.randrange(n)
        st.update(x=_normal(gen, T, K), a=_normal(gen, n, R, K, std=K ** -0.5),
                  b=_normal(gen, n, N, R, std=0.3 * R ** -0.5),
                  scales=torch.rand(n, generator=gen, device=dev) + 0.5, ids=_ints(ids, dev),
                  y=None if case["partial"] else _normal(gen, T, N),
                  indptr=None if case["chunk"] == 1 else _ints(_indptr(lens), dev),
                  max_q=max(lens), of_token=_ints([a for a, q in zip(ids, lens) for _ in range(q)], dev))
    elif case["op"] == "store":
        T, hq, hkv = case["tokens"], case["hq"], case["hkv"]
        nh = hq + 2 * hkv
        # an image or video grid behind some text: the axes' positions differ
        start, w = rng.randrange(0, 4096), 24 + rng.randrange(40)
        i = torch.arange(T, device=dev)
        pos = torch.stack([start + i // (w * w), start + (i // w) % w, start + i % w])
        slots = torch.randperm(T + 64, generator=gen, device=dev)[:T]
        if T > 4:
            slots[rng.randrange(T)] = -1  # a padding token
        pools = T + 64
        st.update(positions=pos.to(torch.int32).contiguous(), slots=slots.to(torch.int32),
                  k_pool=torch.zeros(pools, hkv * HD, dtype=torch.bfloat16, device=dev),
                  v_pool=torch.zeros(pools, hkv * HD, dtype=torch.bfloat16, device=dev),
                  table=_table(dev), qn=_normal(gen, HD, std=0.2).add_(1.0),
                  kn=_normal(gen, HD, std=0.2).add_(1.0),
                  axes=torch.tensor(_axis_map(case), device=dev),
                  sections=(HD // 2 - case["s1"] - case["s2"], case["s1"], case["s2"]))
        if case["parts"]:
            st["parts"] = _normal(gen, case["parts"], T, nh * HD, std=case["parts"] ** -0.5,
                                  dtype=torch.float32)
        else:
            st["qkv"] = _normal(gen, T, nh * HD)
    else:
        lens, hkv = _contexts(case), case["hkv"]
        q_lens = _chunks(case)
        rows, num_pages = _pages(lens, rng, 3)
        st.update(page_table=_ints(rows, dev), seq_lens=_ints(lens, dev), max_seq=max(lens),
                  indptr=None if case["chunk"] == 1 else _ints(_indptr(q_lens), dev),
                  max_q=max(q_lens), k_pool=_keys(gen, num_pages * PAGE, hkv).view(-1, hkv * HD))
        if case["op"] == "bounds":
            st["bounds"] = torch.zeros(num_pages, hkv, 2, HD, dtype=torch.bfloat16, device=dev)
            # (request, logical page) of every page that the new tokens touch
            touched = [(r, p) for r, (n, q) in enumerate(zip(lens, q_lens))
                       for p in range((n - q) // PAGE, (n - 1) // PAGE + 1)]
            st["touched"] = torch.tensor(touched, device=dev)
        else:
            T, hq = sum(q_lens), case["hq"]
            st["v_pool"] = torch.randn(num_pages * PAGE, hkv * HD, generator=gen, device=dev,
                                       dtype=torch.bfloat16)
            paged = st["k_pool"].view(num_pages, PAGE, hkv, HD)
            st["bounds"] = torch.stack([paged.amin(1), paged.amax(1)], 2).contiguous()
            # neighbouring queries of a request look at much the same context
            base = _normal(gen, case["reqs"], hq, HD, dtype=torch.float32)
            of = torch.tensor([r for r, q in enumerate(q_lens) for _ in range(q)], device=dev)
            st["q"] = (0.8 * base[of] + 0.6 * _normal(gen, T, hq, HD, dtype=torch.float32)
                       ).to(torch.bfloat16)
            st["of_token"] = of
            st["at"] = torch.tensor([n - q + i for n, q in zip(lens, q_lens) for i in range(q)],
                                    device=dev)
            st["row"] = torch.tensor([i for q in q_lens for i in range(q)], device=dev)
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    return {"lora": _run_lora, "store": _run_store, "bounds": _run_bounds,
            "sparse": _run_sparse}[st["case"]["op"]](st)


def _run_lora(st):
    case = st["case"]
    if own:
        ops = _ops()
        if "ws" not in st:  # the workspace and the output buffer that a serving loop keeps
            T = st["x"].shape[0]
            st["ws"] = ops.lora_workspace(T, case["k"], case["rank"])
            st["out"] = torch.empty(T, case["n"], device=st["x"].device,
                                    dtype=torch.float32 if case["partial"] else torch.bfloat16)
        keep = dict(q_indptr=st["indptr"], max_q_len=st["max_q"], workspace=st["ws"], out=st["out"])
        if case["partial"]:
            return ops.lora_partial(st["x"], st["a"], st["b"], st["scales"], st["ids"], **keep)
        return ops.lora_add(st["x"], st["a"], st["b"], st["scales"], st["ids"], st["y"], **keep)
    n, R, K = st["a"].shape
    of = st["of_token"].long()
    h = (st["x"].float() @ st["a"].float().view(n * R, K).T).view(-1, n, R)
    pick = of[:, None] == torch.arange(n, device=of.device)  # each token keeps its own adapter's part
    h = (h * (pick * st["scales"])[:, :, None]).view(-1, n * R)
    d = h @ st["b"].float().transpose(1, 2).reshape(n * R, -1)
    return d if case["partial"] else (st["y"].float() + d).to(torch.bfloat16)


def _run_store(st):
    case = st["case"]
    hq, hkv, T = case["hq"], case["hkv"], case["tokens"]
    if own:
        ops = _ops()
        src, call = ((st["parts"], ops.qknorm_mrope_store_kv_partials) if case["parts"]
                     else (st["qkv"], ops.qknorm_mrope_store_kv))
        if "out" not in st:  # kept by a serving loop
            st["out"] = torch.empty(T, hq, HD, dtype=torch.bfloat16, device=src.device)
        q = call(src, st["k_pool"], st["v_pool"], st["positions"], st["slots"], st["table"],
                 st["qn"], st["kn"], hq, hkv, EPS, sections=st["sections"],
                 interleaved=case["interleaved"], out=st["out"])
        return {"q": q, "k_pool": st["k_pool"], "v_pool": st["v_pool"]}
    x = st["parts"].sum(0) if case["parts"] else st["qkv"].float()
    x = x.view(T, hq + 2 * hkv, HD)
    qk, v = x[:, :hq + hkv], x[:, hq + hkv:]
    w = torch.cat([st["qn"].float().expand(hq, HD), st["kn"].float().expand(hkv, HD)])
    qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * w
    at = st["positions"].long()[st["axes"]].T                     # [T, 64]
    pair = torch.arange(HD // 2, device=at.device)
    c, s = st["table"][at, pair][:, None], st["table"][at, pair + HD // 2][:, None]
    lo, hi = qk[..., :HD // 2], qk[..., HD // 2:]
    qk = torch.cat([lo * c - hi * s, lo * s + hi * c], -1).to(torch.bfloat16)
    # a padding token stores nothing: it writes its neighbour's row again
    slots = st["slots"].long()
    src = torch.where(slots >= 0, torch.arange(T, device=at.device), (slots >= 0).long().argmax())
    dst = slots[src]
    st["k_pool"][dst] = qk[src, hq:].reshape(T, -1)
    st["v_pool"][dst] = v[src].reshape(T, -1).to(torch.bfloat16)
    return {"q": qk[:, :hq].contiguous(), "k_pool": st["k_pool"], "v_pool": st["v_pool"]}


def _run_bounds(st):
    hkv = st["case"]["hkv"]
    if own:
        _ops().kv_page_bounds_(st["bounds"], st["k_pool"], st["page_table"], st["seq_lens"], hkv,
                               q_indptr=st["indptr"], max_q_len=st["max_q"])
        return st["bounds"]
    r, p = st["touched"].T
    phys = st["page_table"].long()[r, p]
    k = st["k_pool"].view(-1, PAGE, hkv, HD)[phys].float()
    live = p[:, None] * PAGE + torch.arange(PAGE, device=p.device) < st["seq_lens"][r][:, None]
    live = live[:, :, None, None]
    inf = float("inf")
    st["bounds"][phys] = torch.stack([torch.where(live, k, inf).amin(1),
                                      torch.where(live, k, -inf).amax(1)], 2).to(torch.bfloat16)
    return st["bounds"]


def _run_sparse(st):
    case = st["case"]
    hq, hkv, top = case["hq"], case["hkv"], case["top"]
    if own:
        ops = _ops()
        if "ws" not in st:  # the workspace and the output buffers that a serving loop keeps
            T, dev = st["q"].shape[0], st["q"].device
            st["ws"] = ops.select_pages_workspace(T, st["max_seq"], hkv)
            st["ids"] = torch.empty(T, hkv, top, dtype=torch.int32, device=dev)
            st["out"] = torch.empty(T, hq, HD, dtype=torch.bfloat16, device=dev)
        ids = ops.select_pages(st["q"], st["bounds"], st["page_table"], st["seq_lens"],
                               st["max_seq"], top, hq, hkv, sink_pages=case["sink"],
                               recent_pages=case["recent"], q_indptr=st["indptr"],
                               max_q_len=st["max_q"], workspace=st["ws"], out=st["ids"])
        out = ops.paged_attention_pages(st["q"], st["k_pool"], st["v_pool"], st["page_table"],
                                        st["seq_lens"], ids, hq, hkv, q_indptr=st["indptr"],
                                        max_q_len=st["max_q"], max_seq_len=st["max_seq"],
                                        out=st["out"])
        return {"page_ids": ids, "out": out}
    q, of, at = st["q"], st["of_token"], st["at"]
    T, G, B, n = q.shape[0], hq // hkv, case["reqs"], st["page_table"].shape[1]
    # scores in 64 bits (the choice at the border hangs on them), padded by request
    qp = torch.zeros(B, st["max_q"], hkv, G, HD, dtype=torch.float64, device=q.device)
    qp[of, st["row"]] = q.view(T, hkv, G, HD).double()
    qp = qp.permute(0, 2, 1, 3, 4).reshape(B, hkv, -1, HD)
    bounds = st["bounds"][st["page_table"].long()].permute(0, 2, 3, 4, 1).double()  # [B, hkv, 2, HD, n]
    s = qp.clamp(min=0) @ bounds[:, :, 1] + qp.clamp(max=0) @ bounds[:, :, 0]
    s = s.view(B, hkv, -1, G, n).amax(3).transpose(1, 2)[of, st["row"]]                # [T, hkv, n]
    page = torch.arange(n, device=q.device)
    seen = (at // PAGE + 1)[:, None]
    forced = (page < case["sink"]) | (page >= seen - case["recent"])
    inf = float("inf")
    s = torch.where((page < seen)[:, None], torch.where(forced[:, None], inf, s), -inf)
    best = torch.sort(s, dim=-1, descending=True, stable=True).indices[..., :top]
    best = torch.where(best < seen[..., None], best, n).sort(-1).values
    ids = torch.full((T, hkv, top), -1, dtype=torch.int32, device=q.device)
    ids[..., :best.shape[-1]] = torch.where(best < n, best, -1)
    # attention over the keys of the selected pages
    lid = ids.clamp(min=0).long()
    slot = (st["page_table"].long()[of[:, None, None], lid][..., None] * PAGE
            + torch.arange(PAGE, device=q.device)).view(T, hkv, -1)
    pos = (lid[..., None] * PAGE + torch.arange(PAGE, device=q.device)).view(T, hkv, -1)
    live = (pos <= at[:, None, None]) & (ids >= 0).repeat_interleave(PAGE, -1)
    head = torch.arange(hkv, device=q.device)[:, None]
    k = st["k_pool"].view(-1, hkv, HD)[slot, head].float()
    p = (q.view(T, hkv, G, HD).float() @ k.transpose(2, 3)) * HD ** -0.5
    del k
    p = torch.where(live[:, :, None], p, -inf)
    p = (p - p.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = p @ st["v_pool"].view(-1, hkv, HD)[slot, head].float()
    return {"page_ids": ids, "out": out.to(torch.bfloat16).view(T, hq, HD)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "lora":
        lens = _chunks(case)
        T, K, N, R = sum(lens), case["k"], case["n"], case["rank"]
        used = min(case["adapters"], case["reqs"])
        rows = T * K * 2 + T * N * 4  # x; the fp32 partial, or y and out in bf16
        return {"bytes": rows + used * (K + N) * R * 2, "flops": 2.0 * T * R * (K + N)}
    if case["op"] == "store":
        T, nh = case["tokens"], case["hq"] + 2 * case["hkv"]
        read = T * nh * HD * (4 * case["parts"] if case["parts"] else 2) + T * (HD * 4 + 16)
        return {"bytes": read + T * nh * HD * 2, "flops": 10.0 * T * nh * HD}
    if case["op"] == "bounds":
        pages = sum((n - 1) // PAGE - (n - q) // PAGE + 1
                    for n, q in zip(_contexts(case), _chunks(case)))
        return {"bytes": pages * case["hkv"] * (PAGE + 2) * HD * 2.0,
                "flops": pages * case["hkv"] * PAGE * HD * 2.0}
    hq, hkv, top = case["hq"], case["hkv"], case["top"]
    total, flops = 0.0, 0.0
    for n, q in zip(_contexts(case), _chunks(case)):
        pages = -(-n // PAGE)
        kept = min(top, pages)
        total += q * (hq * HD * 4 + hkv * top * 4) + pages * (hkv * 2 * HD * 2 + 4)
        # the keys and values of the selected pages, each page of a request once
        total += min(pages, q * kept) * hkv * PAGE * HD * 4
        flops += q * hq * (4.0 * HD * kept * PAGE + (4.0 * HD * pages if pages > top else 0.0))
    return {"bytes": total, "flops": flops}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"lora": _exact_lora, "store": _exact_store, "bounds": _exact_bounds,
            "sparse": _exact_sparse}[case["op"]](st)


def _exact_lora(st):
    case = st["case"]
    x = st["x"].double()
    out = x.new_zeros(x.shape[0], case["n"])
    t = 0
    for a, q in zip(st["ids"].tolist(), _chunks(case)):
        if a >= 0:
            h = x[t:t + q] @ st["a"][a].double().T
            out[t:t + q] = (h @ st["b"][a].double().T) * st["scales"][a].double()
        t += q
    return out if case["partial"] else out + st["y"].double()


def _exact_store(st):
    case = st["case"]
    hq, hkv, T = case["hq"], case["hkv"], case["tokens"]
    x = (st["parts"].double().sum(0) if case["parts"] else st["qkv"].double()).view(T, -1, HD)
    q = torch.empty(T, hq, HD, dtype=torch.float64, device=x.device)
    k_pool, v_pool = st["k_pool"].double().view(-1, hkv, HD), st["v_pool"].double().view(-1, hkv, HD)
    keep = st["slots"] >= 0
    for h in range(hq + hkv):
        y = x[:, h] / torch.sqrt((x[:, h] ** 2).sum(1, keepdim=True) / HD + EPS)
        y = y * (st["qn"] if h < hq else st["kn"]).double()
        z = torch.empty_like(y)
        for d, axis in enumerate(_axis_map(case)):
            row = st["table"][st["positions"][axis].long()].double()
            c, s = row[:, d], row[:, d + HD // 2]
            z[:, d] = y[:, d] * c - y[:, d + HD // 2] * s
            z[:, d + HD // 2] = y[:, d] * s + y[:, d + HD // 2] * c
        if h < hq:
            q[:, h] = z
        else:
            k_pool[st["slots"][keep].long(), h - hq] = z[keep]
            v_pool[st["slots"][keep].long(), h - hq] = x[keep, h + hkv]
    return {"q": q, "k_pool": k_pool.view(-1, hkv * HD), "v_pool": v_pool.view(-1, hkv * HD)}


def _exact_bounds(st):
    hkv = st["case"]["hkv"]
    bounds = st["bounds"].double()
    table, keys = st["page_table"].tolist(), st["k_pool"].view(-1, PAGE, hkv, HD)
    lens = st["seq_lens"].tolist()
    for r, p in st["touched"].tolist():
        k = keys[table[r][p], :min(PAGE, lens[r] - p * PAGE)].double()
        bounds[table[r][p], :, 0], bounds[table[r][p], :, 1] = k.min(0).values, k.max(0).values
    return bounds


def _exact_sparse(st):
    case = st["case"]
    hq, hkv, top = case["hq"], case["hkv"], case["top"]
    G, T = hq // hkv, st["q"].shape[0]
    ids = torch.full((T, hkv, top), -1, dtype=torch.int32)
    out = torch.zeros(T, hq, HD, dtype=torch.float64, device=st["q"].device)
    t = 0
    for r, (n, m) in enumerate(zip(_contexts(case), _chunks(case))):
        phys = st["page_table"][r, :-(-n // PAGE)].long()
        slots = (phys[:, None] * PAGE + torch.arange(PAGE, device=phys.device)).view(-1)[:n]
        for h in range(hkv):
            lo, hi = st["bounds"][phys, h, 0].double(), st["bounds"][phys, h, 1].double()
            qh = st["q"][t:t + m, h * G:(h + 1) * G].double()
            key = st["k_pool"].view(-1, hkv, HD)[slots, h].double()
            val = st["v_pool"].view(-1, hkv, HD)[slots, h].double()
            mid, wide = (hi + lo) / 2, (hi - lo) / 2  # max(q lo, q hi) = q mid + |q| wide
            score = (qh @ mid.T + qh.abs() @ wide.T).amax(1).cpu()
            for i in range(m):
                seen = (n - m + i) // PAGE + 1
                first, last = min(case["sink"], seen), max(case["sink"], seen - case["recent"])
                pick = list(range(first)) + list(range(max(first, last), seen))
                if seen <= top:
                    pick = list(range(seen))
                elif top > len(pick):
                    mids = score[i, first:last]
                    order = torch.sort(mids, descending=True, stable=True).indices[:top - len(pick)]
                    pick += [first + j for j in order.tolist()]
                pick.sort()
                ids[t + i, h, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
                at = (torch.tensor(pick)[:, None] * PAGE + torch.arange(PAGE)).view(-1)
                at = at[at <= n - m + i].to(phys.device)
                p = torch.softmax(qh[i] @ key[at].T / math.sqrt(HD), -1)
                out[t + i, h * G:(h + 1) * G] = p @ val[at]
        t += m
    return {"page_ids": ids, "out": out}
