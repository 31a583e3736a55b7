"""The operators of a batched decode step, as cases that can be timed: each in its plain form
(elementary torch operations) and through this library's calls.

    norm      rmsnorm with the residual's addition and a q8_0 output, row by row
    append    RoPE, then q out and k, v into the pages of a cache
    pages     a cache's pages: free, fork and grow (a beam step), and compact
    attention a batch over the pages, sequences of a group sharing their first pages
    adapters  low-rank adapters of many requests added to shared projections

Shapes are the Llama-3.2-1B one (2048 wide, 32 heads of 64 over 8, 16 layers) and a generic
4096-wide one (32 heads of 128 over 8).
"""
import torch

own = False

F16, BF16 = 1, 30           # GGML's type numbers
DTYPE = {F16: torch.float16, BF16: torch.bfloat16}
DEV = "cuda"

_layer = None               # the program's one open layer (own only)


# ---- the cases ------------------------------------------------------------------

def listed():
    return [
        # one token's norm in a decode step
        {"name": "norm 1x2048", "op": "norm", "m": 1, "k": 2048, "add": True},
        # the norms of a long prompt
        {"name": "norm 2048x4096", "op": "norm", "m": 2048, "k": 4096, "add": True},
        # one layer of a decode step of 64 sequences, 1B shape
        {"name": "append 64x1 hd64", "op": "append", "n": 64, "t": 1, "heads": 32, "kv": 8, "hd": 64,
         "page": 16, "type": BF16, "layout": "phd", "max_len": 2048},
        # one layer of four prompts of 1000 tokens
        {"name": "append 4x1000 hd128", "op": "append", "n": 4, "t": 1000, "heads": 32, "kv": 8,
         "hd": 128, "page": 32, "type": F16, "layout": "hpd", "max_len": 1500},
        # a beam step of two requests of four beams, all 16 layers of the 1B shape
        {"name": "beam 2x4", "op": "beam", "parents": 2, "each": 4, "layers": 16, "kv": 8, "hd": 64,
         "page": 16, "type": BF16, "layout": "phd", "max_len": 500, "pages": 512},
        # the same of 32 requests of eight
        {"name": "beam 32x8", "op": "beam", "parents": 32, "each": 8, "layers": 16, "kv": 8, "hd": 64,
         "page": 32, "type": BF16, "layout": "hpd", "max_len": 999, "pages": 1536},
        # a cache half emptied by finished requests, packed to the front
        {"name": "compact 2048", "op": "compact", "seqs": 48, "layers": 16, "kv": 8, "hd": 64,
         "page": 16, "type": BF16, "layout": "phd", "max_len": 600, "pages": 2048},
        # four sequences on a short prompt
        {"name": "attention 4x256", "op": "attention", "n": 4, "groups": 1, "t": 1, "prefix": 256,
         "suffix": 20, "heads": 32, "kv": 8, "hd": 64, "page": 16, "type": BF16, "layout": "phd"},
        # 48 sequences on three prompts, four tokens each to verify
        {"name": "attention 3x16x4 3001", "op": "attention", "n": 48, "groups": 3, "t": 4,
         "prefix": 3001, "suffix": 333, "heads": 32, "kv": 8, "hd": 64, "page": 64, "type": F16,
         "layout": "hpd"},
        # 64 answers on one long document
        {"name": "attention 64x16384 hd128", "op": "attention", "n": 64, "groups": 1, "t": 1,
         "prefix": 16384, "suffix": 512, "heads": 32, "kv": 8, "hd": 128, "page": 32, "type": BF16,
         "layout": "phd"},
        # q, k and v of 16 requests over eight adapters, 1B shape
        {"name": "adapters 16 qkv r16", "op": "adapters", "m": 16, "k": 2048, "ns": "2048,512,512",
         "slots": 8, "rank": 16, "runs": False, "type": BF16},
        # the o projection of prompts of four requests, 2000 rows in all
        {"name": "adapters 2000 r64", "op": "adapters", "m": 2000, "k": 4096, "ns": "4096",
         "slots": 4, "rank": 64, "runs": True, "type": F16},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["norm", "append", "beam", "compact", "attention", "attention", "adapters"])
    page = rng.choice([16, 32, 64, 128])
    kind = {"type": rng.choice([F16, BF16]), "layout": rng.choice(["phd", "hpd"])}
    hd = rng.choice([64, 128])
    if op == "norm":
        k = 32 * _log(rng, 8, 256)
        return {"op": op, "m": _log(rng, 1, max(1, 2048 * 4096 // k)), "k": k, "add": rng.random() < 0.7}
    if op == "append":
        kv, t = rng.choice([1, 2, 4, 8]), _log(rng, 1, 1000)
        return {"op": op, "n": _log(rng, 1, max(1, min(128, 4000 // t))), "t": t,
                "heads": kv * rng.choice([1, 2, 3, 4]), "kv": kv, "hd": hd, "page": page, **kind,
                "max_len": t + _log(rng, 1, 1500)}
    if op == "beam":
        parents, max_len = _log(rng, 1, 32), _log(rng, 8, 999)
        each = rng.randint(1, 8)
        return {"op": op, "parents": parents, "each": each, "layers": rng.randint(1, 16),
                "kv": rng.choice([1, 2, 4, 8]), "hd": 64, "page": page, **kind, "max_len": max_len,
                "pages": parents * (-(-max_len // page) + 2 * each) + rng.randint(1, 200)}
    if op == "compact":
        seqs, max_len = _log(rng, 1, 48), _log(rng, 8, 600)
        return {"op": op, "seqs": seqs, "layers": rng.randint(1, 16), "kv": rng.choice([1, 2, 4, 8]),
                "hd": 64, "page": page, **kind, "max_len": max_len,
                "pages": 2 * seqs * -(-max_len // page) + rng.randint(1, 300)}
    if op == "attention":
        kv, t = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 1, 2, 3, 5, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 7 if kv == 4 else 8 if kv < 4 else 4])
        n = _log(rng, 1, 64)
        most = 64 * 32 * 16384 // (n * heads * t)         # no more work than the largest listed
        return {"op": op, "n": n, "groups": rng.randint(1, min(4, n)), "t": t,
                "prefix": _log(rng, 1, max(2, min(16384, most))), "suffix": _log(rng, t + 1, 512),
                "heads": heads, "kv": kv, "hd": hd, "page": page, **kind}
    rank = rng.choice([4, 8, 16, 24, 32, 64])
    k, ns = rng.choice([(2048, "2048,512,512"), (2048, "8192,8192"), (8192, "2048"), (4096, "4096"),
                        (4096, "4096,1024,1024"), (1280, "1280"), (768, "1000")])
    return {"op": op, "m": _log(rng, 1, 2000 if ns == "4096" else 1000), "k": k, "ns": ns,
            "slots": rng.randint(1, 16), "rank": rank, "runs": rng.random() < 0.5, "type": kind["type"]}


# ---- inputs ---------------------------------------------------------------------

def _pool(gen, c, n_pages, layers):
    """K and V of `layers` layers, seen as [layer][page][position][kv head][hd] whatever the layout."""
    dims = (layers, n_pages, c["page"], c["kv"], c["hd"]) if c["layout"] == "phd" else \
        (layers, n_pages, c["kv"], c["page"], c["hd"])
    kv = [torch.randn(dims, generator=gen, device=DEV, dtype=DTYPE[c["type"]]) for _ in range(2)]
    return kv if c["layout"] == "phd" else [t.transpose(2, 3) for t in kv]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _rope(n_ctx, hd):
    at = torch.arange(n_ctx, dtype=torch.float64)[:, None] * \
        500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)[None]
    return torch.stack((at.cos(), at.sin()), -1).reshape(n_ctx, hd).float().to(DEV)


def _fill_tables(rnd, n_pages, lens, page, n_slots, max_pages, shared=()):
    """Random pages for sequences of these lengths: (table, references). `shared`: for every
    sequence the (key, pages) that it shares with the others of that key, or none."""
    order = torch.randperm(n_pages, generator=rnd).tolist()
    table = torch.zeros(n_slots, max_pages, dtype=torch.int32)
    ref = torch.zeros(n_pages, dtype=torch.int32)
    common = {}
    for s, n in enumerate(lens):
        key, k = shared[s] if shared else (None, 0)
        if k and key not in common:
            common[key] = [order.pop() for _ in range(k)]
        mine = (common[key] if k else []) + [order.pop() for _ in range(-(-n // page) - k)]
        table[s, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
        ref[mine] += 1
    return table.to(DEV), ref.to(DEV)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rnd = torch.Generator().manual_seed(seed)
    draws = lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), generator=rnd).tolist()  # noqa: E731
    normal = lambda *dims: torch.randn(dims, generator=gen, device=DEV)  # noqa: E731
    op, s = c["op"], {"case": c}
    if op == "norm":
        m, k = c["m"], c["k"]
        s["x"] = normal(m, k)
        s["add"] = 0.1 * normal(m, k) if c["add"] else None
        s["w"] = 1 + 0.1 * normal(k)
        s["x_out"] = torch.empty(m, k, device=DEV) if c["add"] else None
        s["q"] = torch.empty(m, k, dtype=torch.int8, device=DEV)
        s["d"] = torch.empty(m, k // 32, device=DEV)
        s["values"] = torch.empty(m, k // 32, 32, dtype=torch.bfloat16, device=DEV)
    elif op == "adapters":
        m, k, slots, rank = c["m"], c["k"], c["slots"], c["rank"]
        s["q"] = torch.randint(-127, 128, (m, k), generator=gen, device=DEV, dtype=torch.int8)
        s["d"] = 0.005 + 0.01 * torch.rand(m, k // 32, generator=gen, device=DEV)
        which = draws(-1, slots - 1, m)
        s["which"] = _ints(sorted(which) if c["runs"] else which)
        s["rank"] = _ints([max(1, rank - r) for r in draws(0, rank // 2, slots)])
        s["scale"] = 0.5 + torch.rand(slots, generator=gen, device=DEV)
        ty = DTYPE[c["type"]]
        s["proj"] = []
        for n in (int(v) for v in c["ns"].split(",")):
            a = (normal(slots, rank, k) * k ** -0.5).to(ty)
            b = (normal(slots, n, rank) * rank ** -0.5).to(ty)
            s["proj"].append((a, b, normal(m, n), torch.empty(m, n, device=DEV)))
    else:
        page = c["page"]
        if op == "append":
            n, t = c["n"], c["t"]
            lens = draws(t, c["max_len"], n)
            n_slots, max_pages = n, -(-c["max_len"] // page)
            n_pages = n * max_pages + 3
            s["qkv"] = [normal(n * t, h * c["hd"]) for h in (c["heads"], c["kv"], c["kv"])]
            s["rope"] = _rope(c["max_len"], c["hd"])
            s["q_out"] = torch.empty(n * t, c["heads"], c["hd"], dtype=DTYPE[c["type"]], device=DEV)
            shared = ()
        elif op == "beam":
            n_slots = c["parents"] * (1 + c["each"])
            lens = draws(max(1, c["max_len"] // 2), c["max_len"], c["parents"])
            max_pages, n_pages, shared = -(-(c["max_len"] + 1) // page), c["pages"], ()
            s["from"] = _ints([p for p in range(c["parents"]) for _ in range(c["each"])])
            s["to"] = _ints(list(range(c["parents"], n_slots)))
        elif op == "compact":
            n_slots, n_pages, shared = c["seqs"], c["pages"], ()
            lens = draws(max(1, c["max_len"] // 2), c["max_len"], n_slots)
            max_pages = -(-c["max_len"] // page)
        else:
            n, g = c["n"], c["groups"]
            cuts = [n * i // g for i in range(g + 1)]
            full = c["prefix"] // page
            pre = [max(0, full - i) for i in range(g)]              # pages that each group shares
            lens = [pre[i] * page + max(1, c["prefix"] - full * page) + draws(c["t"], c["suffix"], 1)[0]
                    for i in range(g) for _ in range(cuts[i + 1] - cuts[i])]
            shared = [(i, pre[i]) for i in range(g) for _ in range(cuts[i + 1] - cuts[i])]
            n_slots, max_pages = n, -(-max(lens) // page)
            n_pages = sum(-(-v // page) for v in lens) - sum((cuts[i + 1] - cuts[i] - 1) * pre[i] for i in range(g)) + 5
            s["slots"], s["group"], s["shared"] = _ints(list(range(n))), _ints(cuts), _ints(pre)
            s["max_len"] = max(lens)
            s["q"] = (2 * normal(n * c["t"], c["heads"], c["hd"])).to(DTYPE[c["type"]])
            s["out"] = torch.empty_like(s["q"])
        s["n_slots"], s["max_pages"], s["n_pages"] = n_slots, max_pages, n_pages
        table, ref = _fill_tables(rnd, n_pages, lens, page, n_slots, max_pages, shared)
        s["meta"] = torch.cat((table.flatten(), ref))               # tables and references in one piece
        s["meta0"] = s["meta"].clone()
        s["table"] = s["meta"][:table.numel()].view(n_slots, max_pages)
        s["ref"] = s["meta"][table.numel():]
        s["len"] = _ints(lens + [0] * (n_slots - len(lens)))
        s["k"], s["v"] = _pool(gen, c, n_pages, c.get("layers", 1))
        if op == "append":
            s["slots"] = _ints(list(range(n_slots)))
        s["live"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    if own:
        _plan(s)
    return s


# ---- the library's calls ----------------------------------------------------------

def _plan(s):
    """The structs and workspaces that a program keeps beside its tensors."""
    global _layer
    from charsiu_b200.lib import AdaptersStruct, AttentionStruct, Layer, PagesStruct
    if _layer is None:
        _layer = Layer(max_k=2048, max_n=2048, max_tensors=1)
    g, c = _layer, s["case"]
    s["layer"] = g
    work = lambda nbytes: torch.zeros(max(1, nbytes), dtype=torch.uint8, device=DEV)  # noqa: E731
    if c["op"] == "adapters":
        s["sets"] = [AdaptersStruct(a=a.data_ptr(), b=b.data_ptr(), rank=s["rank"].data_ptr(),
                                    scale=s["scale"].data_ptr(), k=c["k"], n=b.shape[1],
                                    slots=c["slots"], max_rank=c["rank"], type=c["type"])
                     for a, b, _, _ in s["proj"]]
        s["sets"] = g.adapter_sets(s["sets"])
        s["work"] = work(g.adapters_work(s["sets"], c["m"]))
        s["base_ptrs"] = g.pointers([p[2].data_ptr() for p in s["proj"]])
        s["y_ptrs"] = g.pointers([p[3].data_ptr() for p in s["proj"]])
    elif c["op"] != "norm":
        k = s["k"]
        s["pages"] = PagesStruct(
            k=k.data_ptr(), v=s["v"].data_ptr(), table=s["table"].data_ptr(), len=s["len"].data_ptr(),
            ref=s["ref"].data_ptr(), layer_stride=k.stride(0), page_stride=k.stride(1),
            pos_stride=k.stride(2), head_stride=k.stride(3), type=c["type"], n_layer=k.shape[0],
            n_pages=s["n_pages"], page=c["page"], n_head_kv=c["kv"], head_dim=c["hd"],
            n_seq=s["n_slots"], max_pages=s["max_pages"])
        s["pages_work"] = work(g.pages_work(s["pages"]))
        s["pages"].work = s["pages_work"].data_ptr()
        if c["op"] == "attention":
            s["batch"] = AttentionStruct(
                slots=s["slots"].data_ptr(), group=s["group"].data_ptr(), shared=s["shared"].data_ptr(),
                n_seq=c["n"], n_tok=c["t"], n_head=c["heads"], n_group=c["groups"], max_len=s["max_len"],
                out_type=c["type"], scale=c["hd"] ** -0.5)
            s["work"] = work(g.attention_work(s["pages"], s["batch"]))
            s["batch"].work, s["batch"].work_bytes = s["work"].data_ptr(), s["work"].numel()


def _stream():
    # torch's default stream is CUDA's legacy one (handle 1): 0 would name the layer's own
    return torch.cuda.current_stream().cuda_stream or 1


def _own(s):
    g, c, st = s["layer"], s["case"], _stream()
    op = c["op"]
    if op == "norm":
        add, x_out = s["add"], s["x_out"]
        g.norm_quantise_dev(s["x"].data_ptr(), add.data_ptr() if add is not None else 0,
                            s["w"].data_ptr(), c["m"], c["k"], 1e-5,
                            x_out.data_ptr() if x_out is not None else 0, s["q"].data_ptr(),
                            s["d"].data_ptr(), st)
    elif op == "append":
        q, k, v = s["qkv"]
        g.pages_append_dev(s["pages"], 0, s["slots"].data_ptr(), c["n"], c["t"], c["heads"],
                           q.data_ptr(), k.data_ptr(), v.data_ptr(), s["rope"].data_ptr(),
                           c["max_len"], s["q_out"].data_ptr(), st)
    elif op == "beam":
        n = c["parents"] * c["each"]
        to = s["to"].data_ptr()
        g.pages_free_dev(s["pages"], to, n, st)
        g.pages_fork_dev(s["pages"], s["from"].data_ptr(), to, n, st)
        g.pages_grow_dev(s["pages"], to, n, 1, st)
    elif op == "compact":
        g.pages_compact_dev(s["pages"], s["live"].data_ptr(), st)
    elif op == "attention":
        g.attention_dev(s["pages"], 0, s["batch"], s["q"].data_ptr(), s["out"].data_ptr(), st)
    else:
        g.adapters_dev(s["sets"], c["m"], s["q"].data_ptr(), s["d"].data_ptr(), s["which"].data_ptr(),
                       s["base_ptrs"], s["y_ptrs"], s["work"].data_ptr(), s["work"].numel(), st)


# ---- the plain forms ----------------------------------------------------------------

def _norm(s):
    m, k = s["x"].shape
    x = s["x"] if s["add"] is None else s["x"] + s["add"]
    if s["x_out"] is not None:
        s["x_out"].copy_(x)
    y = x.double()                                        # 64 bits: q is decided next to a border
    v = y * torch.rsqrt((y * y).mean(1, keepdim=True) + 1e-5) * s["w"].double()
    v = v.view(m, k // 32, 32)
    d = v.abs().amax(2) / 127
    inv = torch.where(d > 0, 1 / d, 0.0)
    s["q"].copy_((v * inv[..., None]).round().view(m, k))
    s["d"].copy_(d)


def _append(s):
    c = s["case"]
    n, t, hd, page = c["n"], c["t"], c["hd"], c["page"]
    pos = s["len"].long()[s["slots"].long()][:, None] - t + torch.arange(t, device=DEV)    # [n][t]
    cs = s["rope"][pos].view(n * t, 1, hd // 2, 2)
    q, k, v = (x.view(n * t, -1, hd) for x in s["qkv"])

    def turn(x):
        p = x.view(n * t, -1, hd // 2, 2)
        x0, x1, co, si = p[..., 0], p[..., 1], cs[..., 0], cs[..., 1]
        return torch.stack((x0 * co - x1 * si, x0 * si + x1 * co), -1).view(x.shape)

    at = s["table"].long()[s["slots"].long()[:, None], pos // page].flatten(), (pos % page).flatten()
    s["q_out"].copy_(turn(q))
    s["k"][0][at] = turn(k).to(s["k"].dtype)
    s["v"][0][at] = v.to(s["v"].dtype)


def _free_pages(ref, n):
    return torch.argsort((ref > 0).int(), stable=True)[:n].int()


def _held(s, slots):
    """Which entries of these slots' tables are in use, [n][max_pages]."""
    page = s["case"]["page"]
    used = (s["len"][slots] + page - 1) // page
    return torch.arange(s["max_pages"], device=DEV)[None] < used[:, None]


def _count(s, slots, held, by):
    s["ref"].index_add_(0, s["table"][slots].long().clamp(0, s["n_pages"] - 1).flatten(),
                        torch.where(held, by, 0).int().flatten())


def _beam(s):
    page, table, n_len = s["case"]["page"], s["table"], s["len"]
    to, src = s["to"].long(), s["from"].long()
    n = to.numel()
    _count(s, to, _held(s, to), -1)                       # free
    n_len[to] = 0
    held = _held(s, src)                                  # fork: whole pages shared, the last copied
    filled = n_len[src] % page
    last = (n_len[src] // page).long().clamp(max=s["max_pages"] - 1)
    part = filled > 0
    fresh = _free_pages(s["ref"], n)[(part.int().cumsum(0) - 1).clamp(min=0).long()]
    rows = torch.where(held, table[src], table[to])
    old = table[src, last]
    old_to = rows.gather(1, last[:, None])[:, 0]
    rows.scatter_(1, last[:, None], torch.where(part, fresh, old_to)[:, None])
    table[to] = rows
    n_len[to] = n_len[src]
    _count(s, to, held, 1)
    a, b = torch.where(part, old, 0).long(), torch.where(part, fresh, _free_pages(s["ref"], 1)[0]).long()
    keep = torch.arange(page, device=DEV)[None, :, None, None] < filled[:, None, None, None]
    for pool in (s["k"], s["v"]):
        pool[:, b] = torch.where(keep, pool[:, a], pool[:, b])
    new = n_len[to] % page == 0                           # grow by one token
    fresh = _free_pages(s["ref"], n)[(new.int().cumsum(0) - 1).clamp(min=0).long()]
    at = (n_len[to] // page).long().clamp(max=s["max_pages"] - 1)
    table[to, at] = torch.where(new, fresh, table[to, at])
    s["ref"].index_add_(0, torch.where(new, fresh, 0).long(), new.int())
    n_len[to] += 1


def _compact(s):
    n = s["n_pages"]
    live = s["ref"] > 0
    count = live.sum()
    at = torch.arange(n, device=DEV)
    hole, mover = ~live & (at < count), live & (at >= count)
    # the i-th live page from `count` on goes to the i-th hole below it
    holes = torch.argsort((~hole).int(), stable=True)
    to = torch.where(mover, holes[(mover.int().cumsum(0) - 1).clamp(min=0).long()], at)
    held = _held(s, torch.arange(s["n_slots"], device=DEV))
    s["table"].copy_(torch.where(held, to[s["table"].long()].int(), s["table"]))
    src = torch.nonzero(mover)[:, 0]
    dst = to[src]
    s["ref"][dst] = s["ref"][src]
    s["ref"][src] = 0
    for pool in (s["k"], s["v"]):
        pool[:, dst] = pool[:, src]
    s["live"].copy_(count)


def _attention(s):
    c = s["case"]
    n, t, hd, page, kv = c["n"], c["t"], c["hd"], c["page"], c["kv"]
    slots = s["slots"].long()
    n_len = s["len"].long()[slots]
    at = torch.arange(s["max_len"], device=DEV)
    pages = s["table"].long()[slots][:, at // page]                               # [n][L]
    k, v = (pool[0][pages, at % page].float().transpose(1, 2) for pool in (s["k"], s["v"]))
    q = s["q"].float().view(n, t, kv, -1, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, hd)
    score = torch.matmul(q * hd ** -0.5, k.transpose(2, 3)).view(n, kv, -1, t, s["max_len"])
    seen = at[None, None] <= (n_len[:, None] - t + torch.arange(t, device=DEV))[..., None]   # [n][t][L]
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, kv, -1, s["max_len"]), v).view(n, kv, -1, t, hd)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(n * t, -1, hd))


def _adapters(s):
    c = s["case"]
    m, slots, rank = c["m"], c["slots"], c["rank"]
    x = (s["q"].float().view(m, -1, 32) * s["d"][..., None]).view(m, -1)
    on = (s["which"][:, None] == torch.arange(slots, device=DEV)[None]).float() * s["scale"]        # [m][slots]
    cols = (torch.arange(rank, device=DEV)[None] < s["rank"][:, None]).float()                     # [slots][rank]
    for a, b, base, y in s["proj"]:
        t = torch.matmul(x, a.float().view(slots * rank, -1).t()).view(m, slots, rank)
        t = (t * on[..., None] * cols[None]).view(m, -1)
        torch.add(base, torch.matmul(t, b.float().transpose(1, 2).reshape(slots * rank, -1)), out=y)


def run(state):
    s, op = state, state["case"]["op"]
    if op == "compact":                      # the tables are put back first, so that a pass can be repeated
        s["meta"].copy_(s["meta0"])
    if own:
        _own(s)
    else:
        {"norm": _norm, "append": _append, "beam": _beam, "compact": _compact,
         "attention": _attention, "adapters": _adapters}[op](s)
    return _outputs(s)


def _outputs(s):
    op = s["case"]["op"]
    if op == "norm":
        m, k = s["x"].shape
        torch.mul(s["q"].view(m, k // 32, 32), s["d"][..., None], out=s["values"])
        out = {"values": s["values"], "d": s["d"]}
        return out if s["x_out"] is None else {**out, "x": s["x_out"]}
    if op == "append":
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if op == "beam":
        return {"table": s["table"], "len": s["len"], "ref": s["ref"], "k": s["k"], "v": s["v"]}
    if op == "compact":
        return {"table": s["table"], "ref": s["ref"], "live": s["live"], "k": s["k"], "v": s["v"]}
    return s["out"] if op == "attention" else [p[3] for p in s["proj"]]


# ---- what a pass cannot do without ------------------------------------------------------

def work(case):
    c, op = case, case["op"]
    if op == "norm":
        m, k = c["m"], c["k"]
        return {"bytes": m * k * (13 if c["add"] else 5) + m * k // 8 + 4 * k, "flops": 8 * m * k}
    if op == "append":
        rows, wide = c["n"] * c["t"], (c["heads"] + 2 * c["kv"]) * c["hd"]
        turned = (c["heads"] + c["kv"]) * c["hd"]
        return {"bytes": rows * wide * 6 + min(rows, c["max_len"]) * c["hd"] * 4, "flops": 3 * rows * turned}
    if op in ("beam", "compact"):
        row = 2 * c["layers"] * c["kv"] * c["hd"] * 2            # a position's K and V in all layers
        held = 3 * c["max_len"] // 4 // c["page"] + 1            # pages of a sequence, about
        if op == "beam":
            n = c["parents"] * c["each"]                         # half a page a fork; its table four times
            return {"bytes": n * (row * c["page"] + 24 * held) + 4 * c["pages"], "flops": n * held}
        live = min(c["seqs"] * held, c["pages"])
        moved = live * (c["pages"] - live) // c["pages"]         # live pages behind the live count
        return {"bytes": 2 * moved * row * c["page"] + 16 * c["pages"], "flops": c["pages"]}
    if op == "attention":
        rows = c["n"] * c["t"] * c["heads"]
        keys = c["prefix"] + c["suffix"] // 2
        own_keys = c["n"] * (c["suffix"] // 2) + c["groups"] * c["prefix"]
        return {"bytes": own_keys * c["kv"] * c["hd"] * 4 + rows * c["hd"] * 4, "flops": 4 * rows * keys * c["hd"]}
    ns = [int(v) for v in c["ns"].split(",")]
    m, k, r = c["m"], c["k"], 3 * c["rank"] // 4 + 1
    used = min(m, c["slots"])
    return {"bytes": m * (k + k // 8) + sum(8 * m * n + 2 * used * r * (k + n) for n in ns),
            "flops": sum(2 * m * r * (k + n) for n in ns)}


# ---- the definitions in 64 bits -----------------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c, op = s["case"], s["case"]["op"]
    if op == "norm":
        return _exact_norm(s)
    if op == "append":
        return _exact_append(s)
    if op == "attention":
        return _exact_attention(s)
    if op == "adapters":
        return _exact_adapters(s)
    return _exact_beam(s) if op == "beam" else _exact_compact(s)


def _exact_norm(s):
    x = s["x"].double()
    if s["add"] is not None:
        x = x + s["add"].double()
    rows = (s["x"] if s["add"] is None else s["x"] + s["add"]).double()
    rms = torch.sqrt(torch.einsum("mk,mk->m", rows, rows) / rows.shape[1] + 1e-5)
    v = (rows / rms[:, None] * s["w"].double()).unflatten(1, (-1, 32))
    top = v.abs().max(2).values
    steps = torch.round(127 * v / top[..., None])
    out = {"values": steps * top[..., None] / 127, "d": top / 127}
    return out if s["add"] is None else {**out, "x": x}


def _exact_append(s):
    c = s["case"]
    hd, t = c["hd"], c["t"]
    k, v = s["k"].double(), s["v"].double()
    lens, table = s["len"].tolist(), s["table"].tolist()
    turn = torch.view_as_complex(s["rope"].double().view(-1, hd // 2, 2))
    q_out = []
    for i in range(c["n"]):
        pos = list(range(lens[i] - t, lens[i]))
        rows = slice(i * t, (i + 1) * t)
        z = turn[pos][:, None]

        def rot(x):
            p = torch.view_as_complex(x[rows].double().view(t, -1, hd // 2, 2))
            return torch.view_as_real(p * z).flatten(2)
        q_out.append(rot(s["qkv"][0]))
        pages, at = _ints([table[i][p // c["page"]] for p in pos]).long(), _ints([p % c["page"] for p in pos]).long()
        k[0][pages, at] = rot(s["qkv"][1])
        v[0][pages, at] = s["qkv"][2][rows].double().view(t, -1, hd)
    return {"q": torch.cat(q_out), "k": k, "v": v}


def _exact_beam(s):
    page, n_pages = s["case"]["page"], s["n_pages"]
    table, n_len, ref = s["table"].tolist(), s["len"].tolist(), s["ref"].tolist()
    k, v = s["k"], s["v"]
    lowest = lambda: next(p for p in range(n_pages) if not ref[p])  # noqa: E731
    copies = []
    for a, b in zip(s["from"].tolist(), s["to"].tolist()):
        whole, rest = divmod(n_len[a], page)
        for j in range(whole):
            table[b][j] = table[a][j]
            ref[table[a][j]] += 1
        if rest:
            table[b][whole] = p = lowest()
            ref[p] = 1
            copies.append((table[a][whole], p, rest))
        n_len[b] = n_len[a]
    for b in s["to"].tolist():
        if n_len[b] % page == 0:
            table[b][n_len[b] // page] = p = lowest()
            ref[p] = 1
        n_len[b] += 1
    for a, b, rest in copies:
        k[:, b, :rest] = k[:, a, :rest]
        v[:, b, :rest] = v[:, a, :rest]
    return {"table": _ints(table), "len": _ints(n_len), "ref": _ints(ref), "k": k.double(), "v": v.double()}


def _exact_compact(s):
    page = s["case"]["page"]
    table, n_len, ref = s["table"].tolist(), s["len"].tolist(), s["ref"].tolist()
    k, v = s["k"], s["v"]
    live = sum(r > 0 for r in ref)
    free = (p for p in range(live) if not ref[p])
    moved = {}
    for p in range(live, s["n_pages"]):
        if ref[p]:
            moved[p] = d = next(free)
            ref[d], ref[p] = ref[p], 0
            k[:, d], v[:, d] = k[:, p], v[:, p]
    for row, n in zip(table, n_len):
        for j in range(-(-n // page)):
            row[j] = moved.get(row[j], row[j])
    return {"table": _ints(table), "ref": _ints(ref), "live": _ints([live]), "k": k.double(), "v": v.double()}


def _exact_attention(s):
    c = s["case"]
    t, hd, page, heads = c["t"], c["hd"], c["page"], c["heads"]
    lens = s["len"].tolist()
    out = []
    for i in range(c["n"]):
        n = lens[i]
        pages = s["table"][i, :-(-n // page)].long()
        k, v = (pool[0][pages].flatten(0, 1)[:n].double() for pool in (s["k"], s["v"]))     # [n][kv][hd]
        k, v = (x.repeat_interleave(heads // c["kv"], 1) for x in (k, v))
        q = s["q"][i * t:(i + 1) * t].double()
        w = torch.einsum("thd,nhd->htn", q, k) / hd ** 0.5
        hidden = torch.arange(n, device=DEV)[None] > torch.arange(n - t, n, device=DEV)[:, None]
        out.append(torch.einsum("htn,nhd->thd", w.masked_fill(hidden, -float("inf")).softmax(2), v))
    return torch.cat(out)


def _exact_adapters(s):
    c = s["case"]
    x = s["q"].double() * s["d"].double().repeat_interleave(32, 1)
    out = []
    for a, b, base, _ in s["proj"]:
        y = base.double()
        for i in range(c["slots"]):
            rows = s["which"] == i
            r = int(s["rank"][i])
            y[rows] += float(s["scale"][i]) * (x[rows] @ a[i, :r].double().t() @ b[i, :, :r].double().t())
        out.append(y)
    return out
