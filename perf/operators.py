"""Cases of the serving operators on the paged key/value cache: what they compute and on which sizes they are measured.

Three operators that one step of a server with speculative decoding uses in turn:

``attention``  attention of the newest tokens of a batch whose sequences begin with the same tokens, over a paged
               cache that holds this prefix once
``pages``      copying pages of every layer's pool (a forked sequence's partly filled page, a pool made compact)
``verify``     keeping or replacing drafted tokens by the target's and the draft's probabilities and given random
               numbers

``run`` computes them in a plain form from elementary torch operations, or, where ``own`` is true, by the framework's
entry points. ``exact`` gives the same from the definitions in 64 bits.
"""
import math

import torch

own = False


# ---------------------------------------------------------------------------------------------------- cases
def _attention(name, batch, queries, kv_heads, group, head_dim, block, prefix, tail, padded=0):
    return {"name": name, "op": "attention", "batch": batch, "queries": queries, "kv_heads": kv_heads, "group": group,
            "head_dim": head_dim, "block": block, "prefix": prefix, "tail": tail, "padded": padded}


def _pages(name, layers, num_pages, block, kv_heads, head_dim, moves, partial):
    return {"name": name, "op": "pages", "layers": layers, "num_pages": num_pages, "block": block,
            "kv_heads": kv_heads, "head_dim": head_dim, "moves": moves, "partial": partial}


def _verify(name, batch, drafts, vocab, dtype, ragged, with_draft, pad=0):
    return {"name": name, "op": "verify", "batch": batch, "drafts": drafts, "vocab": vocab, "dtype": dtype,
            "ragged": ragged, "with_draft": with_draft, "pad": pad}


def listed():
    return [
        # a few samples of one prompt with the smallest GPT (12 heads of 64): latency counts
        _attention("attn_gpt_small_4", 4, 1, 12, 1, 64, 16, 512, 64),
        # an ordinary batch behind one system prompt, grouped heads
        _attention("attn_gqa_64", 64, 1, 8, 4, 128, 16, 8192, 512),
        # drafted tokens to be scored: up to 5 queries a sequence, ragged, one padded row, a prefix that ends inside
        # a page; the 16 heads of 128 of the rotary decoder
        _attention("attn_verify_ragged_24", 24, 5, 16, 1, 128, 16, 2051, 300, 1),
        # questions to one long document: few sequences, five query heads to a cached one, pages of 24 tokens
        _attention("attn_document_16", 16, 1, 8, 5, 128, 24, 100003, 1000),
        # many samples with one cached head for all queries
        _attention("attn_mqa_128", 128, 1, 1, 16, 64, 32, 16384, 700),
        # a full server: 256 sequences behind a 32k prompt
        _attention("attn_server_256", 256, 1, 8, 4, 128, 16, 32768, 1024),
        # a prompt forked into 8 samples: the partly filled page of each of 12 layers
        _pages("pages_fork_8", 12, 64, 16, 12, 64, 8, True),
        # 64 sequences forked at once on a larger model
        _pages("pages_fork_64", 24, 256, 16, 8, 128, 64, True),
        # a fragmented pool made compact: a third of its pages move
        _pages("pages_compact_680", 16, 2048, 16, 8, 128, 680, False),
        # one sequence's drafts against the GPT vocabulary
        _verify("verify_one", 1, 4, 50257, "float32", False, True),
        # a batch with ragged drafts, probabilities in bf16 and rows padded as the LM head pads them
        _verify("verify_ragged_64", 64, 5, 50257, "bfloat16", True, True, 47),
        # a large batch and vocabulary
        _verify("verify_256", 256, 8, 131072, "float32", False, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "pages", "verify", "verify"])
    if op == "attention":
        c = _attention("", _log(rng, 1, 256), rng.choice([1, 1, 1, 2, 3, 4, 6, 8]), rng.choice([1, 2, 3, 4, 8, 12, 16]),
                       rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 16]), rng.choice([32, 64, 64, 80, 96, 128, 128, 128]),
                       rng.choice([5, 8, 16, 16, 24, 32, 64, 128]), _log(rng, 16, 131072), _log(rng, 16, 2048))
        c["padded"] = rng.choice([0, 0, 1]) if c["batch"] > 2 else 0

        def cost(c):
            rows = c["batch"] * c["queries"] * c["group"] * c["kv_heads"]
            return max(rows * (c["prefix"] + c["tail"]) * c["head_dim"] / (8192 * 33792 * 128),
                       (c["prefix"] + c["batch"] * c["tail"]) * c["kv_heads"] * c["head_dim"] / (295000 * 1024))

        while cost(c) > 0.8:
            k = rng.choice(["batch", "prefix", "tail"])
            c[k] = max(16 if k != "batch" else 3, int(c[k] * rng.uniform(0.5, 0.9)))
    elif op == "pages":
        c = _pages("", rng.randint(1, 24), _log(rng, 8, 2048), rng.choice([5, 8, 16, 16, 32, 64]),
                   rng.choice([1, 2, 3, 8, 12]), rng.choice([32, 40, 64, 80, 128]), 0, rng.random() < 0.5)
        while c["layers"] * c["num_pages"] * c["block"] * c["kv_heads"] * c["head_dim"] > 16 * 2048 * 16384:
            c["num_pages"] = max(4, c["num_pages"] // 2)
        c["moves"] = _log(rng, 1, max(1, c["num_pages"] // 3))
    else:
        c = _verify("", _log(rng, 1, 256), rng.randint(1, 10), _log(rng, 32, 160000),
                    rng.choice(["float32", "float32", "bfloat16", "float16"]), rng.random() < 0.5,
                    rng.random() < 0.75, rng.choice([0, 0, 3, 64]))
        while c["batch"] * (c["drafts"] + 1) * c["vocab"] > 256 * 9 * 131072:
            c["batch"] = max(1, c["batch"] // 2)
    c.pop("name")
    return c


# ---------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"attention": _prepare_attention, "pages": _prepare_pages, "verify": _prepare_verify}[case["op"]](case, g)


def _randn(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def _pool(k, v, heads, block, head_dim):
    """The framework's pool over tensors that hold the pages."""
    from scirs_b200.inference import KvPageConfig, KvPagePool

    pool = KvPagePool(0, KvPageConfig(block_size=block, num_heads=heads, head_dim=head_dim), "cuda")
    pool.k, pool.v = k, v
    return pool


def _prepare_attention(c, g):
    B, Q, Hkv, G, D, bs, L = (c[k] for k in ("batch", "queries", "kv_heads", "group", "head_dim", "block", "prefix"))
    T = max(c["tail"], Q)
    per = -(-(L + T) // bs)  # pages of the longest chain
    shared = L // bs  # whole pages of the prefix: one copy; a page that it ends in is each sequence's own
    front = -(-L // bs)
    num_pages = front + B * (per - shared) + 3
    ids = torch.randperm(num_pages, device="cuda", generator=g).to(torch.int32)
    k, v = _randn(g, num_pages, bs, Hkv, D), _randn(g, num_pages, bs, Hkv, D)
    prefix_pages = ids[:front].contiguous()
    tables = torch.empty(B, per, dtype=torch.int32, device="cuda")
    tables[:, :shared] = ids[:shared]
    tables[:, shared:] = ids[front:front + B * (per - shared)].view(B, per - shared)
    tail = torch.randint(Q, T + 1, (B,), device="cuda", generator=g)
    tail[0] = Q  # a sequence that has only its newest tokens behind the prefix
    lens = (tail + L).to(torch.int32)
    qlens = torch.randint(1, Q + 1, (B,), device="cuda", generator=g).to(torch.int32) if Q > 1 else None
    if c["padded"]:
        lens[-c["padded"]:] = 0
    q = _randn(g, B, Q, Hkv * G, D, scale=1.5)
    s = dict(case=c, q=q if Q > 1 else q[:, 0].contiguous(), k=k, v=v, prefix_pages=prefix_pages, tables=tables,
             lens=lens, qlens=qlens)
    if own:
        from scirs_b200.inference import PagedAttentionConfig, PagedAttentionForward

        s["pool"] = _pool(k, v, Hkv, bs, D)
        s["attention"] = PagedAttentionForward(PagedAttentionConfig(num_heads=Hkv * G, head_dim=D))
    return s


def _prepare_pages(c, g):
    shape = (c["num_pages"], c["block"], c["kv_heads"], c["head_dim"])
    buf = torch.empty(2 * c["layers"], *shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    perm = torch.randperm(c["num_pages"], device="cuda", generator=g).cpu().to(torch.int32)
    n = c["moves"]
    src, dst = perm[:n].contiguous(), perm[n:2 * n].contiguous()
    counts = None
    if c["partial"]:
        counts = torch.randint(1, c["block"] + 1, (n,), device="cuda", generator=g).cpu().to(torch.int32)
    s = dict(case=c, buf=buf, src=src, dst=dst, counts=counts)
    if own:
        s["pools"] = [_pool(buf[2 * i], buf[2 * i + 1], c["kv_heads"], c["block"], c["head_dim"])
                      for i in range(c["layers"])]
    return s


def _prepare_verify(c, g):
    B, n, V, dt = c["batch"], c["drafts"], c["vocab"], getattr(torch, c["dtype"])
    W = V + c["pad"]
    logits = torch.randn(B, n + 1, W, device="cuda", generator=g) * 3.0
    target = torch.zeros(B, n + 1, W, dtype=dt, device="cuda")[..., :V]
    target.copy_(torch.softmax(logits[..., :V], -1))
    # the draft knows the target's scores up to noise, so that most drafted tokens are kept
    logits = logits[:, :n, :V] + torch.randn(B, n, V, device="cuda", generator=g) * 0.5
    probs = torch.softmax(logits, -1)
    tokens = torch.multinomial(probs.view(B * n, V), 1, generator=g).view(B, n)
    draft = None
    if c["with_draft"]:
        draft = torch.zeros(B, n, W, dtype=dt, device="cuda")[..., :V]
        draft.copy_(probs)
    uniforms = torch.rand(B, n + 1, device="cuda", generator=g)
    lens = torch.randint(0, n + 1, (B,), device="cuda", generator=g).to(torch.int32) if c["ragged"] else None
    return dict(case=c, target=target, draft=draft, tokens=tokens, uniforms=uniforms, lens=lens)


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"attention": _run_attention, "pages": _run_pages, "verify": _run_verify}[state["case"]["op"]](state)


def _run_attention(s):
    if own:
        return s["attention"].forward_shared_prefix(s["q"], s["pool"], s["tables"], s["lens"], s["prefix_pages"],
                                                    s["case"]["prefix"], q_lens=s["qlens"])
    c, k, v, tables, lens = s["case"], s["k"], s["v"], s["tables"], s["lens"].long()
    B, Q, Hkv, G, D, bs, L = (c[x] for x in ("batch", "queries", "kv_heads", "group", "head_dim", "block", "prefix"))
    q = s["q"].float().view(B, Q, Hkv, G, D).permute(2, 0, 1, 3, 4) * D ** -0.5  # [Hkv, B, Q, G, D]
    # how many keys a query sees: query t of a sequence with n of them stands at position length - n + t
    t = torch.arange(Q, device="cuda")
    n = s["qlens"].long()[:, None] if s["qlens"] is not None else Q
    limit = torch.where(t < n, lens[:, None] - n + t + 1, 0)  # [B, Q]
    # the prefix, once for all rows of a cached head
    kp = k[s["prefix_pages"].long()].reshape(-1, Hkv, D)[:L].float().permute(1, 2, 0)  # [Hkv, D, L]
    vp = v[s["prefix_pages"].long()].reshape(-1, Hkv, D)[:L].float().transpose(0, 1)  # [Hkv, L, D]
    sp = (q.reshape(Hkv, B * Q * G, D) @ kp).view(Hkv, B, Q, G, L)
    sp = sp.masked_fill(torch.arange(L, device="cuda") >= limit[None, :, :, None, None], -math.inf)
    # each sequence's own keys
    pos = L + torch.arange(tables.shape[1] * bs - L, device="cuda")
    page = tables.long()[:, pos // bs]  # [B, T]
    kt = k[page, pos % bs].float().permute(2, 0, 3, 1)  # [Hkv, B, D, T]
    vt = v[page, pos % bs].float().permute(2, 0, 1, 3)  # [Hkv, B, T, D]
    st = (q.reshape(Hkv, B, Q * G, D) @ kt).view(Hkv, B, Q, G, -1)
    st = st.masked_fill(pos >= limit[None, :, :, None, None], -math.inf)
    # one softmax over both
    m = torch.maximum(sp.amax(-1, True), st.amax(-1, True)).clamp_min(-1e30)
    sp, st = torch.exp(sp - m), torch.exp(st - m)
    total = sp.sum(-1, True) + st.sum(-1, True)
    o = (sp.view(Hkv, B * Q * G, L) @ vp).view(Hkv, B, Q, G, D)
    o = (o + (st.view(Hkv, B, Q * G, -1) @ vt).view(Hkv, B, Q, G, D)) / total.clamp_min(1e-30)
    o = o.permute(1, 2, 0, 3, 4).reshape(B, Q, Hkv * G, D).to(torch.bfloat16)
    return o if Q > 1 else o[:, 0].contiguous()


def _run_pages(s):
    if own:
        from scirs_b200.inference import copy_pages

        copy_pages(s["pools"], s["src"], s["dst"], counts=s["counts"])
        return s["buf"]
    buf = s["buf"]
    src, dst = s["src"].long().cuda(), s["dst"].long().cuda()
    moved = buf[:, src]
    if s["counts"] is not None:
        full = torch.arange(s["case"]["block"], device="cuda") < s["counts"].cuda()[:, None]
        moved = torch.where(full[None, :, :, None, None], moved, buf[:, dst])
    buf[:, dst] = moved
    return buf


def _run_verify(s):
    if own:
        from scirs_b200.inference import verify_drafts

        return tuple(verify_drafts(s["target"], s["draft"], s["tokens"], s["uniforms"], draft_lens=s["lens"]))
    # whole-number answers that have to hold next to a border: 64 bits throughout
    target, draft, tokens, u = s["target"], s["draft"], s["tokens"], s["uniforms"].double()
    B, n = tokens.shape
    i = torch.arange(n, device="cuda")
    lens = s["lens"].long() if s["lens"] is not None else torch.full((B,), n, device="cuda")
    p = target[:, :n].gather(2, tokens[..., None])[..., 0].double()
    q = draft.gather(2, tokens[..., None])[..., 0].double() if draft is not None else torch.ones_like(p)
    keep = torch.where(q > 0, u[:, :n] * q < p, p > 0) & (i < lens[:, None])
    kept = keep.long().cumprod(1).sum(1)
    b = torch.arange(B, device="cuda")
    # weights of the token to draw: max(p - q, 0) at the first rejection (p where nothing is left), else p
    at = kept.clamp_max(n - 1)  # the place of the first rejection
    w = target[b, kept].double()
    other = draft[b, at].double() if draft is not None else torch.zeros_like(w).scatter_(1, tokens[b, at][:, None], 1.0)
    rest = torch.where((kept < lens)[:, None], (w - other).clamp_min(0.0), w)
    w = torch.where(rest.sum(1, True) > 0, rest, w)
    c = w.cumsum(1)
    drawn = (c <= u[:, n:] * c[:, -1:]).sum(1)
    slot = torch.arange(n + 1, device="cuda")
    out = torch.where(slot < kept[:, None], torch.cat([tokens, tokens[:, :1]], 1), -1)
    out = torch.where(slot == kept[:, None], drawn[:, None], out)
    return kept.to(torch.int32), out


# ---------------------------------------------------------------------------------------------------- what it takes
def work(case):
    c = case
    if c["op"] == "attention":
        B, Q, Hkv, G, D, L = (c[x] for x in ("batch", "queries", "kv_heads", "group", "head_dim", "prefix"))
        live = B - c["padded"]
        tail = (Q + max(c["tail"], Q)) / 2  # on average
        rows = live * (Q + 1) / 2 * Hkv * G if Q > 1 else live * Hkv * G
        return {"bytes": (L + live * tail) * Hkv * D * 4 + 2 * rows * D * 2, "flops": 4 * D * rows * (L + tail)}
    if c["op"] == "pages":
        page = (((1 + c["block"]) / 2) if c["partial"] else c["block"]) * c["kv_heads"] * c["head_dim"] * 2
        return {"bytes": 2 * 2 * c["layers"] * c["moves"] * page, "flops": 0}
    size = torch.finfo(getattr(torch, c["dtype"])).bits // 8
    n = c["drafts"] / 2 if c["ragged"] else c["drafts"]
    rows = 2 - 0.8 ** n if c["with_draft"] else 1  # the draft's row counts where a token is rejected
    return {"bytes": c["batch"] * (rows * c["vocab"] * size + 16 * c["drafts"]), "flops": 3 * c["batch"] * c["vocab"]}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"attention": _exact_attention, "pages": _exact_pages, "verify": _exact_verify}[case["op"]](case, g)


def _exact_attention(c, g):
    """Sequence by sequence over its keys in order: the prefix's pages, then its own."""
    s = _prepare_attention(c, g)
    B, Q, Hkv, G, D, bs, L = (c[x] for x in ("batch", "queries", "kv_heads", "group", "head_dim", "block", "prefix"))
    q = s["q"].view(B, Q, Hkv * G, D)
    out = torch.zeros(B, Q, Hkv * G, D, dtype=torch.float64, device="cuda")
    lens = s["lens"].tolist()
    qlens = s["qlens"].tolist() if s["qlens"] is not None else [Q] * B
    at = torch.arange(L, device="cuda")
    pk, pv = (x[s["prefix_pages"].long()[at // bs], at % bs].double() for x in (s["k"], s["v"]))  # [L, Hkv, D]
    for b in range(B):
        at = torch.arange(L, max(lens[b], L), device="cuda")
        page = s["tables"][b].long()[at // bs]
        own_k, own_v = s["k"][page, at % bs].double(), s["v"][page, at % bs].double()
        for h in range(Hkv):
            keys, values = torch.cat([pk[:, h], own_k[:, h]]), torch.cat([pv[:, h], own_v[:, h]])
            for t in range(qlens[b]):
                seen = lens[b] - qlens[b] + t + 1
                if seen <= 0:
                    continue
                score = q[b, t, h * G:(h + 1) * G].double() @ keys[:seen].T / math.sqrt(D)
                out[b, t, h * G:(h + 1) * G] = torch.softmax(score, -1) @ values[:seen]
    return out if Q > 1 else out[:, 0].contiguous()


def _exact_pages(c, g):
    s = _prepare_pages(c, g)
    buf = s["buf"]
    counts = s["counts"].tolist() if s["counts"] is not None else [c["block"]] * c["moves"]
    for a, b, n in zip(s["src"].tolist(), s["dst"].tolist(), counts):
        buf[:, b, :n] = buf[:, a, :n]
    return buf


def _exact_verify(c, g):
    """Sequence by sequence and draft by draft."""
    s = _prepare_verify(c, g)
    B, n, V = c["batch"], c["drafts"], c["vocab"]
    lens = s["lens"].tolist() if s["lens"] is not None else [n] * B
    kept = torch.zeros(B, dtype=torch.int32)
    out = torch.full((B, n + 1), -1, dtype=torch.int64)
    tokens, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    for b in range(B):
        p = s["target"][b].double()
        for i in range(lens[b] + 1):
            weights = p[i]
            if i == lens[b]:
                break
            x = tokens[b][i]
            if s["draft"] is not None:
                q = s["draft"][b, i].double()
            else:  # a draft without probabilities is certain of its token
                q = torch.zeros_like(weights)
                q[x] = 1.0
            px, qx = float(weights[x]), float(q[x])
            if (px > 0) if qx <= 0 else u[b][i] * qx < px:
                kept[b] += 1
                out[b, i] = x
                continue
            rest = torch.relu(weights - q)
            weights = rest if float(rest.sum()) > 0 else weights
            break
        edges = torch.cumsum(weights, 0)
        out[b, int(kept[b])] = int(torch.searchsorted(edges, edges[-1:] * u[b][n], right=True))
    return kept, out
