"""The paged-cache operators as a user calls them, with their plain forms.

Four operators over one layer's paged key / value cache (pages of 64 positions, a page table
row for each sequence, the layout of the batched token loop):

  append     norms of queries and keys for each head and the rotary position in one pass, the
             key and value rows written into the sequences' pages
  attention  the query tokens of a batch over a prefix that all its sequences share and over
             each sequence's own cache
  weigh      the same attention, which also adds each own position's softmax weight, summed
             over the query heads of its KV head, to the cache's running weights
  evict      brings sequences down to a budget of positions by those weights

`run` computes them with elementary torch operations where `own` is false, and with the
framework's kernels where it is true.  Heads, head sizes, batches, prompt lengths and contexts
are those of the workloads C1 to C5 and of the attention tests.
"""
import math

import torch

own = False

PAGE = 64
EPS = 1e-6
ROPE_BASE = 1_000_000.0
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# the cache that goes with a type of queries: f32 activations keep the framework's f16 cache
CACHE = {"f32": torch.float16, "f16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, type, heads, kv_heads, head_dim, batch, own_min, own_max, prefix=0, tokens_min=1, tokens_max=1, budget=0,
          recent=0):
    c = dict(name=name, op=op, type=type, heads=heads, kv_heads=kv_heads, head_dim=head_dim, batch=batch, own_min=own_min,
             own_max=own_max, prefix=prefix, tokens_min=tokens_min, tokens_max=tokens_max, budget=budget, recent=recent)
    if name is None:
        del c["name"]
    return c


def listed():
    return [
        # one frame of 64 running sequences: the new token of each goes into its cache
        _case("append step", "append", "f32", 32, 8, 128, 64, 128, 1024),
        # the 64 prompts of the batched workload, in one packed batch
        _case("append prompts", "append", "bf16", 32, 8, 128, 64, 0, 0, tokens_min=128, tokens_max=1024),
        # the smallest decode call: one sequence of the tiny model just past its 64-token prompt
        _case("attend short", "attention", "f32", 8, 2, 64, 1, 65, 65),
        # 64 utterances of one voice: a 10 s reference clip (216 frames) with its text, then each one's own text and frames
        _case("attend voice", "attention", "f32", 32, 8, 128, 64, 16, 512, prefix=727),
        # the same voice prompt grown to the 8,192-token prompt of C5, sequences that have just begun
        _case("attend long voice", "attention", "bf16", 32, 8, 128, 64, 1, 256, prefix=8192),
        # a prefix near the model's context, shared by a large batch
        _case("attend longest", "attention", "f16", 32, 8, 128, 128, 1, 64, prefix=32000),
        # 16 texts read behind one voice prompt, ragged
        _case("attend prompts", "attention", "f32", 32, 8, 128, 16, 0, 0, prefix=727, tokens_min=33, tokens_max=400),
        # long prompts behind a shared one
        _case("attend long prompts", "attention", "bf16", 32, 8, 128, 4, 0, 0, prefix=2000, tokens_min=500, tokens_max=2048),
        # a decode step that keeps the running weights, C4's batch in long utterances
        _case("weigh step", "weigh", "f16", 32, 8, 128, 64, 1025, 4096, prefix=216),
        # the last 32 tokens of prompts weigh what to keep of them
        _case("weigh window", "weigh", "bf16", 32, 8, 128, 8, 1968, 8160, tokens_min=32, tokens_max=32),
        # a running batch at its budget: each sequence takes one token in and lets one position go
        _case("turn over", "turnover", "f16", 32, 8, 128, 64, 2048, 2048, budget=2048, recent=512),
        # long prompts brought down to half
        _case("evict half", "evict", "bf16", 32, 8, 128, 16, 6000, 8192, budget=4096, recent=1024),
    ]


SHAPES = [(32, 8, 128), (32, 8, 128), (8, 2, 64), (16, 2, 64), (16, 8, 128), (32, 4, 128), (8, 8, 128), (8, 1, 64)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges, no dearer than the largest listed one."""
    most = max(work(c)["flops"] / 1.6e15 + work(c)["bytes"] / 6.5e12 for c in listed())
    while True:
        op = rng.choice(["append", "attention", "attention", "attention", "weigh", "weigh", "evict", "turnover"])
        heads, kv_heads, head_dim = rng.choice(SHAPES)
        type = rng.choice(["f32", "f16", "bf16"])
        batch = _log(rng, 1, 128)
        own_max = _log(rng, 1, 8192)
        own_min = _log(rng, 1, own_max)
        prefix = tokens = 0
        if op in ("append", "attention", "weigh") and rng.random() < 0.45:
            tokens = _log(rng, 2, 2048 if op != "weigh" else 256)
        if op in ("attention", "weigh") and rng.random() < (0.8 if op == "attention" else 0.4):
            prefix = _log(rng, 1, 32000)
        tokens_min, tokens_max = (rng.randint(1, tokens), tokens) if tokens else (1, 1)
        if tokens and op != "weigh" and rng.random() < 0.5:
            own_min = own_max = 0
        budget = recent = 0
        if op == "evict":
            budget = _log(rng, 1, max(1, own_max))
            recent = rng.randint(0, budget)
        if op == "turnover":
            own_min = own_max
            budget, recent = own_max, rng.randint(1, own_max)
        c = _case(None, op, type, heads, kv_heads, head_dim, batch, own_min, own_max, prefix, tokens_min, tokens_max, budget, recent)
        w = work(c)
        scores = batch * heads * tokens_max * (prefix + own_max + tokens_max)  # what the plain form holds at once
        cached = batch * kv_heads * (own_max + tokens_max) * head_dim
        if w["flops"] / 1.6e15 + w["bytes"] / 6.5e12 <= most and scores <= 1.1e9 and cached <= 7e8 and \
                batch * tokens_max * heads * head_dim <= 4e8:
            return c


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------


def _spread(lo, hi, n):
    """n whole numbers over [lo, hi], both ends among them, in no order."""
    if n == 1:
        return [hi]
    golden = 0.6180339887498949
    at = [0.0, 1.0] + [((i + 1) * golden) % 1.0 for i in range(n - 2)]
    return [lo + int(round(x * (hi - lo))) for x in at]


def _tokens(c):
    """The query tokens of each sequence."""
    return _spread(c["tokens_min"], c["tokens_max"], c["batch"])


def _past(c):
    """What each sequence's cache holds before this call's tokens (before eviction: all that it holds)."""
    return _spread(c["own_min"], c["own_max"], c["batch"])


def _lengths(c):
    if c["op"] in ("append", "turnover") or c["tokens_max"] > 1:
        return [p + t for p, t in zip(_past(c), _tokens(c))]
    return _past(c)


def work(case):
    c = case
    es = 4 if c["type"] == "f32" else 2
    H, G, D, B = c["heads"], c["kv_heads"], c["head_dim"], c["batch"]
    row = 2 * 2 * D  # one position's key and value row of one KV head
    tokens, lengths = _tokens(c), _lengths(c)
    T = sum(tokens)

    def append(T):
        # q, k and v in; q, the two cache rows, position and weight out
        return T * ((H + 2 * G) * D * es + H * D * es + G * row + G * 8 + 4), T * (H + G) * D * 8

    def evict(lengths):
        # weights and positions in; on average the kept rows behind the budget move
        nbytes = 0.0
        for n in lengths:
            if n > c["budget"]:
                tail = n - c["budget"]
                late = min(c["recent"], tail)
                share = (c["budget"] - c["recent"]) / (n - c["recent"])
                nbytes += G * (8 * n + 2 * (late + share * (tail - late)) * (row + 8))
        return nbytes, 0

    if c["op"] == "append":
        nbytes, flops = append(T)
    elif c["op"] == "evict":
        nbytes, flops = evict(lengths)
    elif c["op"] == "turnover":
        nbytes, flops = (x + y for x, y in zip(append(T), evict(lengths)))
    else:
        seen = sum(t * n - t * (t - 1) // 2 for t, n in zip(tokens, lengths))
        nbytes = 2 * T * H * D * es + 4 * T * H + (c["prefix"] + sum(lengths)) * G * row
        if c["op"] == "weigh":
            nbytes += 8 * G * sum(lengths)
        flops = 4 * H * D * (T * c["prefix"] + seen)
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    H, G, D, B = c["heads"], c["kv_heads"], c["head_dim"], c["batch"]
    act, kv = TYPES[c["type"]], CACHE[c["type"]]
    tokens, past, lengths = _tokens(c), _past(c), _lengths(c)
    T = sum(tokens)
    ragged = c["tokens_max"] > 1

    def randn(*shape, dtype, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * scale).to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    max_pages = max(1, -(-max(lengths) // PAGE))
    n_prefix = -(-c["prefix"] // PAGE)
    n_pages = B * max_pages + n_prefix
    order = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    s = {"op": c["op"], "past": ints(past), "lengths": ints(lengths), "prefix_len": c["prefix"],
         "page_table": order[: B * max_pages].view(B, max_pages).contiguous(),
         "prefix_pages": order[B * max_pages:].contiguous() if n_prefix else None,
         "q_start": ints([sum(tokens[:b]) for b in range(B + 1)]) if ragged else None, "most_tokens": c["tokens_max"],
         "budget": c["budget"], "recent": c["recent"]}
    # cached keys: RMS-normed rows with learned gains, so of norm near sqrt(head_dim)
    if c["op"] == "append":
        s["k"], s["v"] = (torch.zeros(n_pages, G, PAGE, D, dtype=kv, device=dev) for _ in range(2))
    else:
        s["k"], s["v"] = (randn(n_pages, G, PAGE, D, dtype=kv) for _ in range(2))
    slots = max_pages * PAGE
    s["positions"] = torch.arange(slots, dtype=torch.int32, device=dev).expand(B, G, slots).contiguous()
    # accumulated weights: a few positions hold most of the mass, one in ten none at all
    mass = torch.rand(B, G, slots, generator=gen, device=dev)
    s["mass"] = torch.where(mass < 0.1, torch.zeros_like(mass), mass.pow(6) * 8.0)
    if c["op"] in ("append", "turnover"):
        s["q_in"], s["k_in"], s["v_in"] = (randn(T, n, D, dtype=act, scale=1.5) for n in (H, G, G))
        s["q_norm"], s["k_norm"] = (1.0 + randn(D, dtype=torch.float32, scale=0.1) for _ in range(2))
        s["pos"] = torch.cat([torch.arange(c["prefix"] + p, c["prefix"] + p + t, dtype=torch.int32) for p, t in zip(past, tokens)]).to(dev)
    elif c["op"] != "evict":
        s["q"] = randn(T, H, D, dtype=act, scale=1.5)
        s["scale"] = 1.0 / math.sqrt(D)
    else:
        s["positions0"], s["mass0"] = s["positions"].clone(), s["mass"].clone()
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def _append_plain(s):
    B, G = s["page_table"].shape[0], s["k"].shape[1]
    T, D = s["q_in"].shape[0], s["q_in"].shape[2]
    dev = s["q_in"].device
    half = torch.arange(0, D, 2, device=dev, dtype=torch.float64)
    angle = s["pos"].double()[:, None] / ROPE_BASE ** (half / D)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, gain):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gain
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)

    q = turned(s["q_in"], s["q_norm"]).to(s["q_in"].dtype)
    start = s["q_start"].long() if s["q_start"] is not None else torch.arange(B + 1, device=dev)
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(start, t, right=True) - 1
    slot = s["past"].long()[seq] + t - start[seq]
    page = s["page_table"].long()[seq, slot // PAGE]
    s["k"][page, :, slot % PAGE] = turned(s["k_in"], s["k_norm"]).to(s["k"].dtype)
    s["v"][page, :, slot % PAGE] = s["v_in"].float().to(s["v"].dtype)
    s["positions"][seq, :, slot] = s["pos"][:, None].expand(T, G)
    s["mass"][seq, :, slot] = 0.0
    s["lengths"].copy_(s["past"] + (start[1:] - start[:-1]).to(torch.int32))
    return q


def _attention_plain(s, weigh):
    q = s["q"]
    T, H, D = q.shape
    B, G = s["page_table"].shape[0], s["k"].shape[1]
    rep, dev = H // G, q.device
    most = s["most_tokens"]
    start = s["q_start"].long() if s["q_start"] is not None else torch.arange(B + 1, device=dev)
    count = start[1:] - start[:-1]
    i = torch.arange(most, device=dev)
    real = i < count[:, None]  # [B][most]
    at = (start[:-1, None] + i).clamp(max=T - 1)
    rows = q.float()[at].view(B, most, G, rep, D).permute(2, 0, 1, 3, 4).reshape(G, B, most * rep, D) * s["scale"]
    pages = s["page_table"].long()
    kv = [x[pages].permute(2, 0, 1, 3, 4).reshape(G, B, -1, D).float() for x in (s["k"], s["v"])]  # [G][B][slots][D]
    n = kv[0].shape[2]
    seen = s["lengths"].long()[:, None] - count[:, None] + i + 1  # [B][most]: a query's own visible positions
    hidden = torch.arange(n, device=dev) >= torch.where(real, seen, 0)[..., None]  # [B][most][slots]
    hidden = hidden[:, :, None].expand(B, most, rep, n).reshape(B, most * rep, n)
    scores = torch.matmul(rows, kv[0].transpose(2, 3)).masked_fill(hidden, -math.inf)
    P = s["prefix_len"]
    if P:
        first = [x[s["prefix_pages"].long()].permute(1, 0, 2, 3).reshape(G, -1, D)[:, :P].float() for x in (s["k"], s["v"])]
        scores = torch.cat((torch.matmul(rows.reshape(G, -1, D), first[0].transpose(1, 2)).view(G, B, most * rep, P), scores), -1)
    top = scores.amax(-1, keepdim=True)
    scores = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = scores.sum(-1, keepdim=True)
    scores = scores / torch.where(total == 0, 1.0, total)
    out = torch.matmul(scores[..., P:], kv[1])
    if P:
        out = out + torch.matmul(scores[..., :P].reshape(G, -1, P), first[1]).view(out.shape)
    lse = (top + torch.log(total)).squeeze(-1)
    if weigh:
        alive = real[:, :, None].expand(B, most, rep).reshape(B, most * rep, 1)
        s["mass"] += (scores[..., P:] * alive).sum(2).permute(1, 0, 2)
    out = out.view(G, B, most, rep, D).permute(1, 2, 0, 3, 4).reshape(B, most, H, D)[real].to(q.dtype)
    lse = lse.view(G, B, most, rep).permute(1, 2, 0, 3).reshape(B, most, H)[real]
    return out, lse


def _evict_plain(s):
    budget, recent = s["budget"], s["recent"]
    n = s["lengths"].long()
    slot = torch.arange(s["mass"].shape[2], device=n.device)
    valid = (slot < n[:, None])[:, None].expand_as(s["mass"])
    newest = s["positions"].masked_fill(~valid, -(2 ** 31)).amax(-1, keepdim=True).long()
    kept_first = valid & (s["positions"].long() > newest - recent)
    by_weight = torch.sort(s["mass"].masked_fill(~valid, -math.inf), dim=-1, descending=True, stable=True).indices
    group = torch.where(kept_first, 0, torch.where(valid, 1, 2))
    order = by_weight.gather(-1, torch.sort(group.gather(-1, by_weight), dim=-1, stable=True).indices)
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order))
    keep = valid & (rank < budget)
    over = (n > budget)[:, None, None]
    to = torch.nonzero(over & ~keep & (slot < budget))  # row by row, slots ascending: as many as there are rows to move
    fro = torch.nonzero(over & keep & (slot >= budget))
    b, g, i, j = to[:, 0], to[:, 1], to[:, 2], fro[:, 2]
    pages = s["page_table"].long()
    s["k"][pages[b, i // PAGE], g, i % PAGE] = s["k"][pages[b, j // PAGE], g, j % PAGE]
    s["v"][pages[b, i // PAGE], g, i % PAGE] = s["v"][pages[b, j // PAGE], g, j % PAGE]
    s["mass"][b, g, i] = s["mass"][b, g, j]
    s["positions"][b, g, i] = s["positions"][b, g, j]
    s["past"].copy_(torch.clamp(s["lengths"], max=budget))


def _cache(s):
    """The framework's cache over the state's buffers: made once, as a program keeps it."""
    if "cache" not in s:
        from fish_s2pro_b200 import PagedKvCache
        s["cache"] = PagedKvCache(s["k"], s["v"], s["page_table"], s["lengths"], positions=s["positions"], mass=s["mass"])
    return s["cache"]


def _append(s):
    if own:
        return _cache(s).append(s["q_in"], s["k_in"], s["v_in"], s["pos"], s["past"], q_start=s["q_start"], q_norm=s["q_norm"],
                                k_norm=s["k_norm"], eps=EPS, rope_base=ROPE_BASE)
    return _append_plain(s)


def _evict(s):
    if own:
        _cache(s).evict(s["budget"], s["recent"], s["past"])
    else:
        _evict_plain(s)


def run(state):
    s = state
    if s["op"] == "append":
        q = _append(s)
        return {"q": q, "k": s["k"], "v": s["v"], "positions": s["positions"], "mass": s["mass"], "lengths": s["lengths"]}
    if s["op"] == "turnover":
        q = _append(s)
        _evict(s)
        s["pos"].add_(1)
        return {"q": q, "k": s["k"], "v": s["v"], "positions": s["positions"], "mass": s["mass"], "past": s["past"]}
    if s["op"] == "evict":
        # a prompt has just been read and weighed: its positions and weights are put in place
        s["positions"].copy_(s["positions0"])
        s["mass"].copy_(s["mass0"])
        _evict(s)
        return {"k": s["k"], "v": s["v"], "positions": s["positions"], "mass": s["mass"], "past": s["past"]}
    weigh = s["op"] == "weigh"
    if own:
        out, lse = _cache(s).attention(s["q"], q_start=s["q_start"], prefix_pages=s["prefix_pages"], prefix_len=s["prefix_len"],
                                       scale=s["scale"], weigh=weigh, return_lse=True)
    else:
        out, lse = _attention_plain(s, weigh)
    return {"out": out, "lse": lse, "mass": s["mass"]} if weigh else {"out": out, "lse": lse}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------


def exact(case, seed):
    c, s = case, prepare(case, seed)

    def append():
        D, B = c["head_dim"], c["batch"]
        table = s["page_table"].cpu()
        tokens, past = _tokens(c), _past(c)
        r = {"q": torch.empty(s["q_in"].shape, dtype=torch.float64, device="cuda"), "k": s["k"].double(), "v": s["v"].double(),
             "positions": s["positions"].clone(), "mass": s["mass"].double()}

        def turn(x, gain, pos):
            x = x.double()
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * gain.double()
            z = torch.view_as_complex(x.view(*x.shape[:-1], D // 2, 2).contiguous())
            freq = torch.exp(-math.log(ROPE_BASE) * torch.arange(D // 2, device=x.device, dtype=torch.float64) * 2 / D)
            z = z * torch.polar(torch.ones_like(freq), pos.double()[:, None] * freq)[:, None]
            return torch.view_as_real(z).reshape(x.shape)

        t0 = 0
        for b in range(B):
            at = slice(t0, t0 + tokens[b])
            t0 += tokens[b]
            pos = s["pos"][at]
            r["q"][at] = turn(s["q_in"][at], s["q_norm"], pos)
            k, v = turn(s["k_in"][at], s["k_norm"], pos), s["v_in"][at].double()
            done = 0
            while done < tokens[b]:
                slot = past[b] + done
                m = min(PAGE - slot % PAGE, tokens[b] - done)
                page, first = int(table[b, slot // PAGE]), slot % PAGE
                r["k"][page, :, first:first + m] = k[done:done + m].transpose(0, 1)
                r["v"][page, :, first:first + m] = v[done:done + m].transpose(0, 1)
                done += m
            r["positions"][b, :, past[b]:past[b] + tokens[b]] = pos
            r["mass"][b, :, past[b]:past[b] + tokens[b]] = 0
        r["lengths"] = torch.tensor([p + t for p, t in zip(past, tokens)], dtype=torch.int32)
        return r

    def evict(r, table, lengths):
        """Evicts in r (k, v, positions, mass) row by row."""
        budget = c["budget"]
        pos, mass = r["positions"].cpu().tolist(), r["mass"].cpu().tolist()
        for b in range(c["batch"]):
            n = lengths[b]
            if n <= budget:
                continue
            for g in range(c["kv_heads"]):
                p, w = pos[b][g][:n], mass[b][g][:n]
                edge = max(p) - c["recent"]
                kept = set(sorted(range(n), key=lambda j: (p[j] <= edge, -w[j], j))[:budget])
                holes = [j for j in range(budget) if j not in kept]
                tail = [j for j in range(budget, n) if j in kept]
                if not holes:
                    continue
                to, fro = (torch.tensor(x, device=table.device) for x in (holes, tail))
                for x in ("k", "v"):
                    r[x][table[b, to // PAGE], g, to % PAGE] = r[x][table[b, fro // PAGE], g, fro % PAGE]
                for x in ("positions", "mass"):
                    r[x][b, g, to] = r[x][b, g, fro]
        r["past"] = torch.tensor([min(n, budget) for n in lengths], dtype=torch.int32)

    def attention(weigh):
        H, G, D, P = c["heads"], c["kv_heads"], c["head_dim"], c["prefix"]
        rep = H // G
        table = s["page_table"].long()
        tokens, lengths = _tokens(c), _lengths(c)
        T = sum(tokens)
        out = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
        lse = torch.full((T, H), -math.inf, dtype=torch.float64, device="cuda")
        mass = s["mass"].double()
        t0 = 0
        for b in range(c["batch"]):
            n, t = lengths[b], tokens[b]
            for g in range(G):
                def rows(x):
                    mine = x[table[b], g].reshape(-1, D)[:n]
                    return (torch.cat((x[s["prefix_pages"].long(), g].reshape(-1, D)[:P], mine)) if P else mine).double()

                k, v = rows(s["k"]), rows(s["v"])
                q = s["q"][t0:t0 + t, g * rep:(g + 1) * rep].double()
                x = torch.einsum("thd,nd->thn", q, k) * s["scale"]
                last = P + n - t + torch.arange(t, device=x.device)  # the last position that a query sees
                x.masked_fill_((torch.arange(P + n, device=x.device) > last[:, None])[:, None], -math.inf)
                lse[t0:t0 + t, g * rep:(g + 1) * rep] = torch.logsumexp(x, -1)
                w = torch.softmax(x, -1).nan_to_num(0.0)
                out[t0:t0 + t, g * rep:(g + 1) * rep] = torch.einsum("thn,nd->thd", w, v)
                if weigh:
                    mass[b, g, :n] += w[..., P:].sum((0, 1))
            t0 += t
        return {"out": out, "lse": lse, "mass": mass} if weigh else {"out": out, "lse": lse}

    if c["op"] == "append":
        return append()
    if c["op"] == "turnover":
        r = append()
        evict(r, s["page_table"].long(), r.pop("lengths").tolist())
        return r
    if c["op"] == "evict":
        r = {"k": s["k"].double(), "v": s["v"].double(), "positions": s["positions"].clone(), "mass": s["mass"].double()}
        evict(r, s["page_table"].long(), _lengths(c))
        return r
    return attention(c["op"] == "weigh")
